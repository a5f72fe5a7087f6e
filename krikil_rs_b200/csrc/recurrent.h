// Host-side launchers of the recurrent layers over state slots (short causal
// convolution, selective state space scan) and of the log probabilities
// (internal C++ interface; the argument checks live in capi_recurrent.cu).
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace krk {

// Where a call's requests keep their states: request s continues from slot
// init[s] (below 0: from nothing) and leaves its state in slot slots[s].
struct SlotArgs {
    void* state; int64_t stride; int num_slots;  // state == nullptr: from nothing, and nothing is kept
    const int32_t* slots;                        // nullptr: slot s
    const int32_t* init;                         // nullptr: the slot that it goes to
};

constexpr int CONV_MAX_WIDTH = 4;
struct ConvArgs {
    const void* x; int64_t x_st;                 // (t, c) at t*x_st + c
    const float* w; const float* bias;           // [C][W], [C] or nullptr
    void* out; int64_t o_st;
    SlotArgs slot;                               // [num_slots][W-1][C] of x's type
    const int32_t* cu;                           // [S+1]; nullptr: one row a request
    int T, S, C;
    bool silu;
    bool aligned;                                // w on 16 bytes (the launcher's own)
};
cudaError_t causal_conv(const ConvArgs& a, int W, int type, cudaStream_t s);

constexpr int SCAN_MAX_STATES = 256;
constexpr int SCAN_THREADS = 128;
constexpr int SCAN_BLOCKS = 4;  // blocks a multiprocessor, by registers
constexpr int SCAN_LANE = 16;   // states a lane holds, if there are as many
constexpr int SCAN_ALONE = 5;   // a request of up to so many pieces is not split
constexpr int SCAN_PIECE = 64;  // fewest rows of one
struct ScanArgs {
    const void* x; int64_t x_st;                 // (t, d) at t*x_st + d
    const void* dt; int64_t dt_st;
    const void* z; int64_t z_st;                 // nullptr: no gate
    const void* b; int64_t b_st, b_sg;           // (t, g, n) at t*b_st + g*b_sg + n
    const void* c; int64_t c_st, c_sg;
    void* out; int64_t o_st;
    const float* a;                              // [D][N]
    const float* d; const float* dt_bias;        // [D] or nullptr
    SlotArgs slot;                               // [num_slots][D][N] float32
    const int32_t* cu;                           // [S+1]; nullptr: one row a request
    int T, S, D, N, G;
};
// How the scan is launched: with scratch of scan_work_floats floats, requests of
// more than SCAN_ALONE * rows rows are walked in pieces of that many (rows 0: none).
struct ScanPlan {
    int rows;
    bool thin;  // lanes of few states
};
ScanPlan scan_plan(int T, int S, int D, int N, int G, int max_len);
size_t scan_work_floats(int T, int D, int N, int G, int max_len);
constexpr int64_t scan_split_room(int64_t T, int rows) { return T / rows * (SCAN_ALONE + 1) / SCAN_ALONE + 2; }
cudaError_t selective_scan(const ScanArgs& a, int type, int max_len, float* work, cudaStream_t s);
cudaError_t selective_step(const ScanArgs& a, int type, cudaStream_t s);

constexpr int LOGPROBS_MAX_TOP = 32;
struct LogprobArgs {
    const void* logits; int64_t ld; int R, V;    // (r, v) at r*ld + v
    const int32_t* tokens; int K;                // [R][K]
    float* lp;                                   // [R][K]
    float* entropy;                              // [R] or nullptr
    int top;
    int32_t* top_ids; float* top_lp;             // [R][top]
};
cudaError_t token_logprobs(const LogprobArgs& a, int type, cudaStream_t s);

// Whether a tensor whose rows are `stride` elements apart can be accessed so many bytes at a time.
inline bool fits(const void* p, int64_t stride, size_t bytes, size_t elem) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && stride * (int64_t)elem % (int64_t)bytes == 0;
}

}  // namespace krk
