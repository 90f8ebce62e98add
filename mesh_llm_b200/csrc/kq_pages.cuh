// The paged key / value cache as its kernels see it: geometry, who owns a row of a ragged batch, rotation.
//
// A pool holds pages [n_pages][n_kv][page][hd], keys and values in one pool each; table[s][i] names the page of positions
// i page .. (i + 1) page - 1 of sequence s.  An entry outside 0 .. n_pages - 1, or a position past the table's end, is a position
// that is not there: it is neither stored nor seen.  Row r of a call belongs to the sequence s with
// row_start[s] <= r < row_start[s + 1] and stands at position pos0[s] + r - row_start[s]; a sequence with pos0 < 0 has no positions.
//
// e4m3 pages: the 16 positions of an aligned block share one scale 2^e per head, -15 <= e <= 7, in scale[page][n_kv][page / 16].  A power
// of two costs a floating code nothing and makes a rescaled code exact above e4m3's smallest normal number; within these exponents
// every code times its scale is an f16 number, so attention works on exactly what the page stands for.
#pragma once
#include "kq_common.cuh"

#include <cuda_bf16.h>

constexpr int KQ_PAGE_BLOCK = 16;
constexpr int64_t KQ_MOST_ELEMENTS = (int64_t)1 << 48; // of a pool or of a call's rows with what lies between them: more than any device holds

struct KqPages {
    uint8_t *k, *v;
    float *ks, *vs;
    const int32_t *table;
    int64_t n_pages, page_bytes; // bytes from one page to the next
    int32_t table_len, table_stride, page, n_kv;
};
struct KqBatch {
    const int32_t *row_start, *pos0;
    int32_t rows, n_seq;
};
struct KqTurns { // turns per position of each rotated pair in units of 2^-64; on = 0: keys and queries are used as they come
    uint64_t f[64];
    int32_t on, neox;
};

// checks of a b200_kv_pages and its batch that need no device memory (kq_pages_append.cu)
b200_status kq_pages_check(const char *who, const b200_kv_pages *c, const b200_page_batch *b, KqPages *out, KqBatch *batch);
b200_status kq_rows_check(const char *who, const char *what, const void *p, uint32_t type, int64_t rows, int64_t stride, int64_t width);
KqTurns kq_turns(float theta, int neox, int hd);
// memory from the first byte of a buffer to behind its last
struct KqSpan {
    const char *what = "";
    uintptr_t from = 0, to = 0;
    KqSpan() {}
    KqSpan(const char *what, const void *p, int64_t bytes) : what(what), from((uintptr_t)p), to(from + bytes) {}
    bool over(const KqSpan &x) const { return from < x.to && x.from < to; }
};
inline KqSpan kq_rows_span(const char *what, const void *p, int64_t es, int64_t rows, int64_t stride, int64_t width) { return KqSpan(what, p, ((rows - 1) * stride + width) * es); }
// the cache's pools (and scales) against a buffer of the call
b200_status kq_pages_apart(const char *who, const b200_kv_pages *c, const KqSpan &x);

#ifdef __CUDACC__
// cos and sin of pos * f turns, f in units of 2^-64: the product's low 64 bits are the angle within its turn, as exact as f is (5.5e-15 of it, kq_turns: 10^-10
// turns at position 10^5, where 32 bits would leave 0.01).  Its first 24 bits are exact in f32, the next 24 are put back to first order, the rest is cut off.
__device__ __forceinline__ float2 kq_turn(uint64_t f, int pos) {
    const uint64_t x = f * (uint64_t)(uint32_t)pos;
    const float t = (float)((int32_t)(x >> 32) >> 8) * 1.1920929e-7f /* 2^-23: half turns */, d = (float)((uint32_t)(x >> 16) & 0xffffffu) * (6.2831853f * 3.5527137e-15f /* 2^-48 */);
    float s, c;
    sincospif(t, &s, &c);
    return make_float2(fmaf(-s, d, c), fmaf(c, d, s));
}
// first and past-the-last row of sequence s, inside the call's rows whatever row_start holds
__device__ __forceinline__ int2 kq_seq_rows(const KqBatch &b, int s) {
    const int lo = min(max(b.row_start[s], 0), b.rows), hi = min(max(b.row_start[s + 1], lo), b.rows);
    return make_int2(lo, hi);
}
// page of sequence s that holds position pos, -1: not there
__device__ __forceinline__ int kq_page_of(const KqPages &c, int s, int64_t pos) {
    const int64_t i = pos / c.page;
    if (pos < 0 || i >= c.table_len) return -1;
    const int id = c.table[(int64_t)s * c.table_stride + i];
    return id >= 0 && id < c.n_pages ? id : -1;
}
__device__ __forceinline__ uint16_t kq_e4m3x2(float lo, float hi) { // round to nearest, beyond +-448 to that, NaN stays
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
// four codes as two pairs of f16 (halves of a register as they are: no shift to reach the upper two)
__device__ __forceinline__ void kq_e4m3x4_h2(uint32_t w, uint32_t &lo, uint32_t &hi) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
}
// two numbers as f16, and what that leaves of them
__device__ __forceinline__ uint32_t kq_h2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t kq_h2_low(float a, float b, uint32_t hi) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
    return kq_h2(a - f.x, b - f.y);
}
__device__ __forceinline__ float kq_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// largest of a warp's values, none of them negative: their bits are in order
__device__ __forceinline__ float kq_warp_top(float v) { return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v))); }
// activations as f32
template <typename T> __device__ __forceinline__ float2 kq_ld2(const T *p);
template <> __device__ __forceinline__ float2 kq_ld2<float>(const float *p) { return *reinterpret_cast<const float2 *>(p); }
template <> __device__ __forceinline__ float2 kq_ld2<__half>(const __half *p) { return __half22float2(*reinterpret_cast<const __half2 *>(p)); }
template <> __device__ __forceinline__ float2 kq_ld2<__nv_bfloat16>(const __nv_bfloat16 *p) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(p));
}
template <typename T> __device__ __forceinline__ float kq_ld1(const T *p) { return (float)*p; }
__device__ __forceinline__ void kq_st2_type(uint32_t type, void *p, int64_t at, float a, float b) {
    if (type == B200_TYPE_F32) *reinterpret_cast<float2 *>((float *)p + at) = make_float2(a, b);
    else if (type == B200_TYPE_F16) *reinterpret_cast<__half2 *>((__half *)p + at) = __floats2half2_rn(a, b);
    else *reinterpret_cast<__nv_bfloat162 *>((__nv_bfloat16 *)p + at) = __floats2bfloat162_rn(a, b);
}
#endif
