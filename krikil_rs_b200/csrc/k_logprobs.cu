// Log probabilities of given tokens, the entropy and the best alternatives of
// each row of logits: with m the row's maximum and s = sum e^(x - m),
//   lp(i) = (x_i - m) - log s,   H = log s - sum e^(x - m) (x - m) / s.
#include "kernels.h"
#include "recurrent.cuh"

namespace krk {
namespace {

constexpr int LP_THREADS = 256, LP_WARPS = LP_THREADS / 32;
constexpr float kLog2e = 1.44269504088896341f, kLowest = -3.402823466e38f;

// The order of the alternatives as whole numbers: larger logits first, of equal
// ones the lower index; NaN counts as -inf and -0 as 0.
KRK_DEV unsigned long long order_key(float x, int i) {
    x = x == x ? x + 0.0f : -INFINITY;
    const unsigned u = __float_as_uint(x);
    return (unsigned long long)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (0xffffffffu - (unsigned)i);
}

template <typename V, typename F>
KRK_DEV V block_fold(V x, V* part, F fold) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x = fold(x, __shfl_xor_sync(0xffffffffu, x, o));
    __syncthreads();  // part may still be read
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = x;
    __syncthreads();
    x = part[0];
#pragma unroll
    for (int w = 1; w < LP_WARPS; ++w) x = fold(x, part[w]);
    return x;
}

// (x - m) - log s; a row that its mask leaves empty gives every token -inf.
KRK_DEV float log_prob(float x, float m, float s) { return s == 0.0f ? -INFINITY : (x - m) - logf(s); }

template <typename T>
__global__ void __launch_bounds__(LP_THREADS) logprobs_kernel(LogprobArgs a) {
    __shared__ float part[LP_WARPS];
    __shared__ unsigned long long keys[LP_WARPS];
    const int row = blockIdx.x, tid = threadIdx.x;
    const T* x = (const T*)a.logits + row * a.ld;
    float m = kLowest;
    for (int i = tid; i < a.V; i += LP_THREADS) m = fmaxf(m, to_f32(x[i]));
    m = block_fold(m, part, [](float p, float q) { return fmaxf(p, q); });
    float s = 0.0f, e = 0.0f;
    for (int i = tid; i < a.V; i += LP_THREADS) {
        const float u = to_f32(x[i]) - m, p = fast_exp2(u * kLog2e);
        s += p;
        e = fmaf(p, fmaxf(u, -1000.0f), e);  // 0 times -inf is 0 here
    }
    const auto add = [](float p, float q) { return p + q; };
    s = block_fold(s, part, add);
    e = block_fold(e, part, add);
    if (a.entropy && tid == 0) a.entropy[row] = s == 0.0f ? 0.0f : logf(s) - e / s;
    for (int k = tid; k < a.K; k += LP_THREADS) {
        const int id = a.tokens[(int64_t)row * a.K + k];
        if (id >= a.V) check_fail(CHK_TOKEN);
        a.lp[(int64_t)row * a.K + k] = id < 0 ? 0.0f : id >= a.V ? -INFINITY : log_prob(to_f32(x[id]), m, s);
    }
    unsigned long long before = ~0ull;
    for (int k = 0; k < a.top; ++k) {
        unsigned long long best = 0;
        for (int i = tid; i < a.V; i += LP_THREADS) {
            const unsigned long long key = order_key(to_f32(x[i]), i);
            if (key < before && key > best) best = key;
        }
        before = block_fold(best, keys, [](unsigned long long p, unsigned long long q) { return p > q ? p : q; });
        if (tid == 0) {
            const int id = (int)(0xffffffffu - (unsigned)before);
            a.top_ids[(int64_t)row * a.top + k] = id;
            a.top_lp[(int64_t)row * a.top + k] = log_prob(to_f32(x[id]), m, s);
        }
    }
}

}  // namespace

cudaError_t token_logprobs(const LogprobArgs& a, int type, cudaStream_t s) {
    if (type == 0)
        logprobs_kernel<float><<<a.R, LP_THREADS, 0, s>>>(a);
    else if (type == 1)
        logprobs_kernel<__half><<<a.R, LP_THREADS, 0, s>>>(a);
    else
        logprobs_kernel<__nv_bfloat16><<<a.R, LP_THREADS, 0, s>>>(a);
    add_launches(1);
    return cudaGetLastError();
}

}  // namespace krk
