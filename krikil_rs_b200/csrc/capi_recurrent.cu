// C entry points of the recurrent layers over state slots (k_causal_conv.cu,
// k_selective.cu) and of the log probabilities (k_logprobs.cu): argument
// checks, then the launchers.  Nothing is launched by a refused call.
#include <cuda_runtime.h>

#include <string>

#include "../../include/krikil_cuda.h"
#include "recurrent.h"

namespace krk {
int report_error(int status, const std::string& msg);  // capi.cu: sets krk_last_error()
}

namespace {

int invalid(const char* who, const char* msg) {
    return krk::report_error(KRK_INVALID, std::string(who) + ": " + msg);
}

int done(const char* who, cudaError_t e) {
    if (e == cudaSuccess) return KRK_OK;
    return krk::report_error(e == cudaErrorInvalidValue ? KRK_INVALID : KRK_CUDA,
                             std::string(who) + ": " + cudaGetErrorString(e));
}

int elem_size(int type) { return type == KRK_TYPE_F32 ? 4 : type == KRK_TYPE_F16 || type == KRK_TYPE_BF16 ? 2 : 0; }

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// A tensor [T, width] that is read: rows may lie anywhere.
bool readable(const void* p, int es) { return p && aligned(p, es); }
// One that is written: its rows may not overlap.
bool writable(const void* p, int64_t stride, int64_t rows, int64_t width, int es) {
    return p && aligned(p, es) && (rows <= 1 || stride >= width);
}

// Whether two tensors [rows, p_w] and [rows, q_w] share memory.
bool overlap(const void* p, int64_t p_st, int64_t p_w, const void* q, int64_t q_st, int64_t q_w, int64_t rows, int es) {
    if (rows <= 0) return false;
    const int64_t a = (int64_t)(uintptr_t)p, b = (int64_t)(uintptr_t)q, pr = p_st * es, qr = q_st * es;
    const auto low = [&](int64_t at, int64_t row) { return row < 0 ? at + (rows - 1) * row : at; };
    const auto high = [&](int64_t at, int64_t row, int64_t w) { return (row > 0 ? at + (rows - 1) * row : at) + w * es; };
    if (high(a, pr, p_w) <= low(b, qr) || high(b, qr, q_w) <= low(a, pr)) return false;
    if (rows > 1 && pr == qr && pr > 0) {  // columns of one matrix are apart if each begins behind the other's end
        const int64_t off = ((a - b) % pr + pr) % pr;
        return off < q_w * es || pr - off < p_w * es;
    }
    return true;
}

// Whether the scan's output shares memory with an input [T][D] that it is not.
bool over_input(const krk::ScanArgs& a, const void* p, int64_t st, int es) {
    const bool same = p == a.out && (a.T <= 1 || st == a.o_st);
    return p && !same && overlap(a.out, a.o_st, a.D, p, st, a.D, a.T, es);
}
// And with B or C [T][G][N]: with what they span, then, if it does, with one of their groups.
bool over_groups(const krk::ScanArgs& a, const void* p, int64_t st, int64_t sg, int es) {
    const int64_t reach = (a.G - 1) * sg;
    const char* first = (const char*)p;
    if (!overlap(a.out, a.o_st, a.D, first + (reach < 0 ? reach * es : 0), st, a.N + (reach < 0 ? -reach : reach), a.T, es))
        return false;
    for (int g = 0; g < a.G; ++g)
        if (overlap(a.out, a.o_st, a.D, first + g * sg * es, st, a.N, a.T, es)) return true;
    return false;
}

const char* slots_fault(const krk::SlotArgs& a, int64_t size, int es) {
    if (!a.state) return a.slots || a.init || a.num_slots ? "slots and init need a state" : nullptr;
    if (a.num_slots <= 0) return "num_slots must be positive";
    if (!aligned(a.state, es)) return "state must be aligned to its elements";
    if (a.num_slots > 1 && a.stride < size) return "the slots' stride is shorter than a state";
    return nullptr;
}

}  // namespace

extern "C" {

static int conv_call(const char* who, const krk::ConvArgs& a, int W, int type, cudaStream_t stream) {
    const int es = elem_size(type);
    if (!es) return invalid(who, "unknown element type");
    if (W < 2 || W > krk::CONV_MAX_WIDTH) return invalid(who, "the width must be 2, 3 or 4");
    if (a.T < 0 || a.S < 0 || a.C <= 0 || a.C > (1 << 24))
        return invalid(who, "rows and requests must not be negative, channels 1 to 2^24");
    if (const char* f = slots_fault(a.slot, (int64_t)(W - 1) * a.C, es)) return invalid(who, f);
    if (a.S == 0) return KRK_OK;
    if (!a.w || !aligned(a.w, 4) || !aligned(a.bias, 4)) return invalid(who, "weight and bias must be set (bias may be null) and aligned");
    if (a.T > 0 && (!readable(a.x, es) || !writable(a.out, a.o_st, a.T, a.C, es)))
        return invalid(who, "x and out must be set and aligned to their elements, rows of out must not overlap");
    if (overlap(a.x, a.x_st, a.C, a.out, a.o_st, a.C, a.T, es)) return invalid(who, "out must not overlap x");
    return done(who, krk::causal_conv(a, W, type, stream));
}

int krk_k_causal_conv(void* x, int64_t x_st, const float* weight, const float* bias, void* out, int64_t o_st, int type,
                      void* state, int64_t state_stride, int num_slots, const int32_t* slots, const int32_t* init,
                      const int32_t* cu, int T, int S, int C, int W, int silu, void* stream) {
    const char* who = "causal_conv";
    if (!cu) return invalid(who, "null pointer");
    const krk::ConvArgs a{x, x_st, weight, bias, out, o_st, {state, state_stride, num_slots, slots, init}, cu, T, S, C,
                          silu != 0, false};
    return conv_call(who, a, W, type, (cudaStream_t)stream);
}

int krk_k_causal_conv_step(void* x, int64_t x_st, const float* weight, const float* bias, void* out, int64_t o_st,
                           int type, void* state, int64_t state_stride, int num_slots, const int32_t* slots,
                           const int32_t* init, int B, int C, int W, int silu, void* stream) {
    const char* who = "causal_conv_step";
    if (!state) return invalid(who, "null pointer");
    const krk::ConvArgs a{x, x_st, weight, bias, out, o_st, {state, state_stride, num_slots, slots, init}, nullptr, B,
                          B, C, silu != 0, false};
    return conv_call(who, a, W, type, (cudaStream_t)stream);
}

static int scan_call(const char* who, const krk::ScanArgs& a, int type, int max_len, float* work, size_t work_floats,
                     cudaStream_t stream) {
    const int es = elem_size(type);
    if (!es) return invalid(who, "unknown element type");
    if (a.T < 0 || a.S < 0) return invalid(who, "rows and requests must not be negative");
    if (a.N < 1 || a.N > krk::SCAN_MAX_STATES) return invalid(who, "N must be 1 to 256");
    if (a.G < 1 || a.D < 1 || a.D > (1 << 24) || a.D % a.G) return invalid(who, "D must be 1 to 2^24 and a multiple of G");
    if (const char* f = slots_fault(a.slot, (int64_t)a.D * a.N, 4)) return invalid(who, f);
    if (a.S == 0) return KRK_OK;
    if (!a.a || !aligned(a.a, 4) || !aligned(a.d, 4) || !aligned(a.dt_bias, 4))
        return invalid(who, "a must be set, and a, d and dt_bias aligned");
    if (a.T > 0 && (!readable(a.x, es) || !readable(a.dt, es) || !readable(a.b, es) || !readable(a.c, es) ||
                    (a.z && !readable(a.z, es)) || !writable(a.out, a.o_st, a.T, a.D, es)))
        return invalid(who, "x, dt, b, c and out must be set and aligned to their elements, rows of out must not overlap");
    if (over_input(a, a.x, a.x_st, es) || over_input(a, a.dt, a.dt_st, es) || over_input(a, a.z, a.z_st, es) ||
        over_groups(a, a.b, a.b_st, a.b_sg, es) || over_groups(a, a.c, a.c_st, a.c_sg, es))
        return invalid(who, "out must be x, dt or z with their strides, or not overlap them, and not overlap b and c");
    if (!a.cu) return done(who, krk::selective_step(a, type, stream));
    if (max_len < 0) return invalid(who, "max_len must not be negative");
    const size_t need = krk::scan_work_floats(a.T, a.D, a.N, a.G, max_len);
    if (need > 0 && (!work || work_floats < need || !aligned(work, 16)))
        return krk::report_error(KRK_INVALID, std::string(who) + ": work must be 16-byte aligned and hold " +
                                                  std::to_string(need) + " floats");
    return done(who, krk::selective_scan(a, type, max_len, work, stream));
}

size_t krk_selective_scan_work_floats(int T, int D, int N, int G, int max_len) {
    if (T <= 0 || D <= 0 || N <= 0 || N > krk::SCAN_MAX_STATES || G <= 0 || D % G || max_len < 0) return 0;
    return krk::scan_work_floats(T, D, N, G, max_len);
}

int krk_k_selective_scan(void* x, int64_t x_st, void* dt, int64_t dt_st, void* z, int64_t z_st, void* b, int64_t b_st,
                         int64_t b_sg, void* c, int64_t c_st, int64_t c_sg, void* out, int64_t o_st, int type,
                         const float* a, const float* d, const float* dt_bias, float* state, int64_t state_stride,
                         int num_slots, const int32_t* slots, const int32_t* init, const int32_t* cu, int T, int S,
                         int D, int N, int G, int max_len, float* work, size_t work_floats, void* stream) {
    const char* who = "selective_scan";
    if (!cu) return invalid(who, "null pointer");
    const krk::ScanArgs s{x, x_st, dt, dt_st, z, z_st, b, b_st, b_sg, c, c_st, c_sg, out, o_st, a, d, dt_bias,
                          {state, state_stride, num_slots, slots, init}, cu, T, S, D, N, G};
    return scan_call(who, s, type, max_len, work, work_floats, (cudaStream_t)stream);
}

int krk_k_selective_step(void* x, int64_t x_st, void* dt, int64_t dt_st, void* z, int64_t z_st, void* b, int64_t b_st,
                         int64_t b_sg, void* c, int64_t c_st, int64_t c_sg, void* out, int64_t o_st, int type,
                         const float* a, const float* d, const float* dt_bias, float* state, int64_t state_stride,
                         int num_slots, const int32_t* slots, const int32_t* init, int B, int D, int N, int G,
                         void* stream) {
    const char* who = "selective_step";
    if (!state) return invalid(who, "null pointer");
    const krk::ScanArgs s{x, x_st, dt, dt_st, z, z_st, b, b_st, b_sg, c, c_st, c_sg, out, o_st, a, d, dt_bias,
                          {state, state_stride, num_slots, slots, init}, nullptr, B, B, D, N, G};
    return scan_call(who, s, type, 0, nullptr, 0, (cudaStream_t)stream);
}

int krk_k_token_logprobs(void* logits, int64_t ld, int type, int R, int V, const int32_t* tokens, int K,
                         float* logprobs, float* entropy, int top, int32_t* top_ids, float* top_logprobs,
                         void* stream) {
    const char* who = "token_logprobs";
    const int es = elem_size(type);
    if (!es) return invalid(who, "unknown element type");
    if (R < 0 || V < 1 || V > (1 << 30) || K < 0) return invalid(who, "R and K must not be negative, V 1 to 2^30");
    if (top < 0 || top > krk::LOGPROBS_MAX_TOP || top > V) return invalid(who, "top must be 0 to 32 and at most V");
    if (R == 0) return KRK_OK;
    if (!logits || !aligned(logits, es)) return invalid(who, "logits must be set and aligned to their elements");
    if ((K > 0 && (!tokens || !logprobs)) || (top > 0 && (!top_ids || !top_logprobs))) return invalid(who, "null pointer");
    const krk::LogprobArgs a{logits, ld, R, V, tokens, K, logprobs, entropy, top, top_ids, top_logprobs};
    return done(who, krk::token_logprobs(a, type, (cudaStream_t)stream));
}

}  // extern "C"
