// C entry points of the paged key-value cache: argument checks, then the
// launchers of k_paged_kv.cu and of the attention (paged_attn.cuh, with its
// engines in k_paged_attn_f32.cu, k_paged_attn_f16.cu and k_paged_attn_bf16.cu).
// Nothing is launched by a refused call.
#include <cuda_runtime.h>

#include <cmath>
#include <string>

#include "../../include/krikil_cuda.h"
#include "paged.h"

namespace krk {
int report_error(int status, const std::string& msg);  // capi.cu: sets krk_last_error()
}

namespace {

int invalid(const char* who, const std::string& msg) {
    return krk::report_error(KRK_INVALID, std::string(who) + ": " + msg);
}

int done(const char* who, cudaError_t e) {
    if (e == cudaSuccess) return KRK_OK;
    return krk::report_error(e == cudaErrorInvalidValue ? KRK_INVALID : KRK_CUDA,
                             std::string(who) + ": " + cudaGetErrorString(e));
}

int log2_exact(int n) {  // -1: not a power of two
    for (int i = 0; i < 31; ++i)
        if (n == (1 << i)) return i;
    return -1;
}

int elem_size(int type) { return type == KRK_TYPE_F32 ? 4 : type == KRK_TYPE_F16 || type == KRK_TYPE_BF16 ? 2 : 0; }

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

struct Dim {
    int64_t size, stride;  // the stride of a dimension of one element does not matter
};

// Four elements at a time: the pointer and every stride.
bool vec4(const void* p, int size, std::initializer_list<Dim> dims) {
    if (!p || !aligned(p, 4 * size)) return false;
    for (const Dim& d : dims)
        if (d.size > 1 && (d.stride < 0 || d.stride % 4)) return false;
    return true;
}

// Written memory: a dimension of more than one element steps over whole heads.
bool distinct(int dh, std::initializer_list<Dim> dims) {
    for (const Dim& d : dims)
        if (d.size > 1 && d.stride < dh) return false;
    return true;
}

// Checks that the pool and the table are addressable; returns "" or what is wrong.
std::string pool_fault(int num_pages, int page_size, int width) {
    const int shift = log2_exact(page_size);
    if (shift < 0 || page_size > 65536) return "page_size must be a power of two of at most 65536";
    if (num_pages <= 0 || ((int64_t)num_pages << shift) > INT32_MAX)
        return "num_pages must be positive and num_pages * page_size below 2^31";
    if (width <= 0 || ((int64_t)width << shift) > (1 << 30))
        return "the table's width must be positive and width * page_size at most 2^30";
    return "";
}

std::string types_fault(int type, int cache_type) {
    if (!elem_size(type) || !elem_size(cache_type)) return "unknown element type";
    if (type != cache_type && type != KRK_TYPE_F32) return "a 16-bit q needs a cache of the same type";
    return "";
}

}  // namespace

extern "C" {

int krk_k_kv_page_plan(const int32_t* new_tokens, const int32_t* lens, int32_t* table, int64_t table_ld, int B,
                       int width, const int32_t* free_pages, const int32_t* free_count, int num_pages, int page_size,
                       int32_t* lens_out, int32_t* free_count_out, int32_t* cu_new, int32_t* positions,
                       int32_t* slots, int rows, int32_t* status, void* stream) {
    const char* who = "kv_page_plan";
    const std::string f = pool_fault(num_pages, page_size, width);
    if (!f.empty()) return invalid(who, f);
    if (B <= 0 || rows < 0) return invalid(who, "B must be positive and rows not negative");
    if (table_ld < width) return invalid(who, "table_ld is shorter than the table's width");
    if (!new_tokens || !lens || !table || !free_pages || !free_count || !lens_out || !free_count_out || !cu_new ||
        !status || (rows > 0 && (!positions || !slots)))
        return invalid(who, "null pointer");
    const krk::PagePlanArgs a{new_tokens, lens, table, table_ld, B, width, free_pages, free_count, num_pages,
                              log2_exact(page_size), lens_out, free_count_out, cu_new, positions, slots, rows, status};
    return done(who, krk::kv_page_plan(a, (cudaStream_t)stream));
}

int krk_k_kv_page_release(const uint8_t* done_mask, const int32_t* lens, const int32_t* table, int64_t table_ld,
                          int B, int width, int32_t* free_pages, const int32_t* free_count, int num_pages,
                          int page_size, int32_t* lens_out, int32_t* free_count_out, int32_t* status, void* stream) {
    const char* who = "kv_page_release";
    const std::string f = pool_fault(num_pages, page_size, width);
    if (!f.empty()) return invalid(who, f);
    if (B <= 0) return invalid(who, "B must be positive");
    if (table_ld < width) return invalid(who, "table_ld is shorter than the table's width");
    if (!done_mask || !lens || !table || !free_pages || !free_count || !lens_out || !free_count_out || !status)
        return invalid(who, "null pointer");
    const krk::PageReleaseArgs a{done_mask, lens, table, table_ld, B, width, free_pages, free_count, num_pages,
                                 log2_exact(page_size), lens_out, free_count_out, status};
    return done(who, krk::kv_page_release(a, (cudaStream_t)stream));
}

int krk_k_rope_kv_append_paged(void* q, int64_t q_st, int64_t q_sh, void* k, int64_t k_st, int64_t k_sh, void* v,
                               int64_t v_st, int64_t v_sh, int type, void* q_out, int64_t qo_st, int64_t qo_sh,
                               void* kc, void* vc, int64_t c_sp, int64_t c_st, int64_t c_sh, int cache_type,
                               const int32_t* slots, const int32_t* positions, int T, int Hq, int Hkv, int dh,
                               int rot_dim, int num_pages, int page_size, float theta, void* stream) {
    const char* who = "rope_kv_append_paged";
    const std::string f = pool_fault(num_pages, page_size, 1), g = types_fault(type, cache_type);
    if (!f.empty()) return invalid(who, f);
    if (!g.empty()) return invalid(who, g);
    if (T < 0 || Hq < 0 || Hkv <= 0 || Hq > 65535 || Hkv > 65535)
        return invalid(who, "T and Hq must not be negative, Hkv positive, heads at most 65535");
    if (dh < 4 || dh > 256 || dh % 4) return invalid(who, "dh must be a multiple of 4 of at most 256");
    if (rot_dim < 0 || rot_dim > dh || rot_dim % 2) return invalid(who, "rot_dim must be even and at most dh");
    if (!(theta > 0.f) || !std::isfinite(theta)) return invalid(who, "theta must be positive and finite");
    if (T == 0) return KRK_OK;
    const int es = elem_size(type), cs = elem_size(cache_type);
    if (!vec4(k, es, {{T, k_st}, {Hkv, k_sh}}) || !vec4(v, es, {{T, v_st}, {Hkv, v_sh}}) ||
        !vec4(kc, cs, {{num_pages, c_sp}, {page_size, c_st}, {Hkv, c_sh}}) ||
        !vec4(vc, cs, {{num_pages, c_sp}, {page_size, c_st}, {Hkv, c_sh}}) ||
        (Hq > 0 && (!vec4(q, es, {{T, q_st}, {Hq, q_sh}}) || !vec4(q_out, es, {{T, qo_st}, {Hq, qo_sh}}))))
        return invalid(who, "pointers must be set and aligned to four elements, strides multiples of four");
    if (!distinct(dh, {{num_pages, c_sp}, {page_size, c_st}, {Hkv, c_sh}}) ||
        (Hq > 0 && !distinct(dh, {{T, qo_st}, {Hq, qo_sh}})))
        return invalid(who, "strides of the caches and q_out must not be shorter than dh");
    if (!slots || !positions) return invalid(who, "null pointer");
    const int shift = log2_exact(page_size);
    const krk::RopeAppendArgs a{q, q_st, q_sh, k, k_st, k_sh, v, v_st, v_sh, q_out, qo_st, qo_sh, kc, vc, c_sp, c_st,
                                c_sh, slots, positions, T, Hq, Hkv, dh, rot_dim, shift, (int64_t)num_pages << shift,
                                krk::rope_turns(rot_dim, theta)};
    return done(who, krk::rope_kv_append_paged(a, type, cache_type, (cudaStream_t)stream));
}

size_t krk_attn_paged_work_floats(int B, int Hq, int Hkv, int dh, int max_len, int window) {
    if (B <= 0 || Hkv <= 0 || Hq < Hkv || Hq % Hkv || dh < 4 || dh > 256 || dh % 4 || max_len < 0 || window < 0)
        return 0;
    return krk::attn_paged_work_floats(B, Hq, Hkv, dh, max_len, window);
}

int krk_k_attn_decode_paged(void* q, int64_t q_sb, int64_t q_sh, int type, void* kc, void* vc, int64_t c_sp,
                            int64_t c_st, int64_t c_sh, int cache_type, const int32_t* table, int64_t table_ld,
                            int width, int num_pages, int page_size, const int32_t* lens, int B, int Hq, int Hkv,
                            int dh, float scale, int window, int max_len, void* out, int64_t o_sb, int64_t o_sh,
                            float* lse, float* work, size_t work_floats, void* stream) {
    const char* who = "attn_decode_paged";
    const std::string f = pool_fault(num_pages, page_size, width), g = types_fault(type, cache_type);
    if (!f.empty()) return invalid(who, f);
    if (!g.empty()) return invalid(who, g);
    if (B < 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || Hq > 65535 || (int64_t)B * Hq > INT32_MAX)
        return invalid(who, "B must not be negative, Hq a positive multiple of Hkv of at most 65535, B * Hq below 2^31");
    if (dh < 4 || dh > 256 || dh % 4) return invalid(who, "dh must be a multiple of 4 of at most 256");
    if (!std::isfinite(scale * 1.44269504088896341f)) return invalid(who, "scale (times log2(e)) must be finite");
    if (window < 0 || max_len < 0) return invalid(who, "window and max_len must not be negative");
    if (table_ld < width) return invalid(who, "table_ld is shorter than the table's width");
    if (B == 0) return KRK_OK;
    const int es = elem_size(type), cs = elem_size(cache_type);
    if (!vec4(q, es, {{B, q_sb}, {Hq, q_sh}}) || !vec4(out, es, {{B, o_sb}, {Hq, o_sh}}) ||
        !vec4(kc, cs, {{num_pages, c_sp}, {page_size, c_st}, {Hkv, c_sh}}) ||
        !vec4(vc, cs, {{num_pages, c_sp}, {page_size, c_st}, {Hkv, c_sh}}))
        return invalid(who, "pointers must be set and aligned to four elements, strides multiples of four");
    if (!distinct(dh, {{B, o_sb}, {Hq, o_sh}})) return invalid(who, "strides of out must not be shorter than dh");
    if (!table || !lens) return invalid(who, "null pointer");
    const int shift = log2_exact(page_size);
    const int64_t cap = (int64_t)width << shift;
    const int bound = (int)(max_len > 0 && max_len < cap ? max_len : cap);
    const size_t need = krk::attn_paged_work_floats(B, Hq, Hkv, dh, bound, window);
    if (need > 0 && (!work || work_floats < need || !aligned(work, 16)))
        return invalid(who, "work must be 16-byte aligned and hold " + std::to_string(need) + " floats");
    // (the engines choose by the strides, and a dimension of one element has none)
    if (num_pages == 1) c_sp = 0;
    if (page_size == 1) c_st = 0;
    if (Hkv == 1) c_sh = 0;
    const krk::PagedAttnArgs a{q, q_sb, q_sh, kc, vc, c_sp, c_st, c_sh, table, table_ld, width, num_pages, shift,
                               lens, B, Hq, Hkv, dh, scale, window,
                               bound, out, o_sb, o_sh, lse, work, work ? work_floats : 0};
    return done(who, krk::attn_decode_paged(a, type, cache_type, (cudaStream_t)stream));
}

}  // extern "C"
