// Host-side launchers of the paged key-value cache kernels (internal C++
// interface; the argument checks live in capi_paged.cu).
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace krk {

// Multiprocessors of the current device, 0 if that cannot be read.
int paged_sm_count();

enum ElemType { ELEM_F32 = 0, ELEM_F16 = 1, ELEM_BF16 = 2 };  // KRK_TYPE_*

// Status bits of the page planner and the release (KRK_PAGES_*).
enum PageStatus : int {
    PAGES_EXHAUSTED = 1,
    PAGES_ROW_FULL = 2,
    PAGES_ROWS = 4,
    PAGES_BAD_LENGTH = 8,
    PAGES_OVERFLOW = 16,
};

struct PagePlanArgs {
    const int32_t* new_tokens; const int32_t* lens;  // [B]
    int32_t* table; int64_t table_ld; int B, width;  // table[b*table_ld + i], i < width
    const int32_t* free_pages; const int32_t* free_count;
    int num_pages, page_shift;                       // page size 1 << page_shift
    int32_t* lens_out; int32_t* free_count_out;
    int32_t* cu_new;                                 // [B+1]
    int32_t* positions; int32_t* slots; int rows;    // [rows]
    int32_t* status;
};
cudaError_t kv_page_plan(const PagePlanArgs& a, cudaStream_t s);

struct PageReleaseArgs {
    const uint8_t* done; const int32_t* lens;
    const int32_t* table; int64_t table_ld; int B, width;
    int32_t* free_pages; const int32_t* free_count;
    int num_pages, page_shift;
    int32_t* lens_out; int32_t* free_count_out;
    int32_t* status;
};
cudaError_t kv_page_release(const PageReleaseArgs& a, cudaStream_t s);

// RoPE turns per position, theta^(-2i/rot) / (2 pi) for pair i, in 64 bits.
constexpr int ROPE_PAGED_PAIRS = 128;
struct RopeTurns {
    double f[ROPE_PAGED_PAIRS];
};
RopeTurns rope_turns(int rot_dim, double theta);

struct RopeAppendArgs {
    const void* q; int64_t q_st, q_sh;               // (t,h,d) at t*q_st + h*q_sh + d
    const void* k; int64_t k_st, k_sh;
    const void* v; int64_t v_st, v_sh;
    void* q_out; int64_t qo_st, qo_sh;
    void* kc; void* vc; int64_t c_sp, c_st, c_sh;    // (page,slot,h,d) at page*c_sp + slot*c_st + h*c_sh + d
    const int32_t* slots; const int32_t* positions;  // [T]
    int T, Hq, Hkv, dh, rot;
    int page_shift; int64_t num_slots;               // num_pages << page_shift
    RopeTurns turns;
};
cudaError_t rope_kv_append_paged(const RopeAppendArgs& a, int act, int cache, cudaStream_t s);

struct PagedAttnArgs {
    const void* q; int64_t q_sb, q_sh;
    const void* kc; const void* vc; int64_t c_sp, c_st, c_sh;
    const int32_t* table; int64_t table_ld; int width, num_pages, page_shift;
    const int32_t* lens;
    int B, Hq, Hkv, dh;
    float scale;
    int window;                                      // 0: every key
    int max_len;                                     // a bound of the lengths that the launch is sized for
    void* out; int64_t o_sb, o_sh;
    float* lse;                                      // [B][Hq] or nullptr
    float* work;                                     // of work_floats, nullptr when clusters take the call
    size_t work_floats;
};
size_t attn_paged_work_floats(int B, int Hq, int Hkv, int dh, int max_len, int window);
cudaError_t attn_decode_paged(const PagedAttnArgs& a, int act, int cache, cudaStream_t s);

}  // namespace krk
