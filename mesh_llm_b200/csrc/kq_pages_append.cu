// New keys and values into the pages of their sequences, the keys rotated on the way (b200_kv_pages_append).
//
// One CTA takes the new rows that fall into one aligned block of 16 positions of one sequence: it works out their cosines and
// sines once, then a warp takes a head's keys and values, a lane the same 2 or 4 dimensions of every row, all rows' loads in flight
// together.  An e4m3 block is one warp's own, so its scale (the smallest power of two that brings the largest of the new values to
// at most 448, never less than the scale of rows the block holds already) needs no atomics and does not depend on timing;
// rows it holds are rescaled in place when the scale grows.
//
// What no attention may meet behind a mask stays out of the values: a value beyond the page type's range goes in as the largest
// one (f16 65504, e4m3 448 * 2^7), and a NaN in v goes in as 0 with a NaN at its place in the token's k, so that every query that
// sees the token gets NaN and no other does.
#include "kq_pages.cuh"

#include <math.h>

namespace {

constexpr int WARPS = 8; // heads of a CTA

struct Rows {
    const void *k, *v;
    int64_t k_stride, v_stride;
    uint32_t type;
};

// the sequence of row r: how many of row_start[1 .. n_seq] are at or below it; every lane of a warp takes part
__device__ __forceinline__ int seq_of_row(const int32_t *row_start, int n_seq, int r, int lane) {
    int lo = 0, hi = n_seq; // the answer is in [lo, hi]
    while (hi - lo > 0) {
        const int n = hi - lo, step = (n + 31) / 32, at = lo + min(n, (lane + 1) * step);
        const unsigned below = __ballot_sync(0xffffffffu, row_start[at] <= r);
        const int full = __popc(below & ~(below + 1)); // leading lanes whose row starts at or before r
        const int nlo = lo + min(n, full * step);
        hi = full == 32 ? nlo : min(hi, nlo + step - 1);
        lo = nlo;
    }
    return lo;
}

__device__ __forceinline__ float clamp_to(float x, float m) { // NaN stays
    x = x > m ? m : x;
    return x < -m ? -m : x;
}

template <int HD, bool F8, int N, bool SPLIT> struct Block {
    static constexpr int P = HD / 64; // pairs of dimensions that a lane holds of each row
    static constexpr bool split = SPLIT; // pairs are (i, i + HD / 2), else (2 i, 2 i + 1)

    // dimension of the lane's element e (0 .. 2 P - 1)
    __device__ static int dim(int e, int lane) {
        if (!split) return 2 * P * lane + e;
        return HD == 128 ? (e >> 1) * 64 + 2 * lane + (e & 1) : e * 32 + lane;
    }
    __device__ static void load(float (&x)[N][2 * P], const Rows &r, const void *p, int64_t at, int64_t stride, int cnt, int lane) {
#pragma unroll
        for (int j = 0; j < N; j++) {
            if (j >= cnt) {
#pragma unroll
                for (int e = 0; e < 2 * P; e++) x[j][e] = 0.f;
                continue;
            }
            const int64_t o = at + j * stride;
            if (HD == 64 && split) {
                x[j][0] = kq_ld1_type(r.type, p, o + lane);
                x[j][1] = kq_ld1_type(r.type, p, o + 32 + lane);
                continue;
            }
#pragma unroll
            for (int u = 0; u < P; u++) {
                const float2 t = kq_ld2_type(r.type, p, o + dim(2 * u, lane));
                x[j][2 * u] = t.x;
                x[j][2 * u + 1] = t.y;
            }
        }
    }
    // rows off .. off + cnt - 1 of the block at `page` (its first code) and `scale`
    __device__ static void store(float (&x)[N][2 * P], uint8_t *page, float *scale, int off, int cnt, int lane) {
        if constexpr (!F8) {
#pragma unroll
            for (int j = 0; j < N; j++) {
                if (j >= cnt) continue;
                __half *row = (__half *)page + (off + j) * HD;
                if (HD == 64 && split) {
                    row[lane] = __float2half_rn(clamp_to(x[j][0], 65504.f));
                    row[32 + lane] = __float2half_rn(clamp_to(x[j][1], 65504.f));
                    continue;
                }
#pragma unroll
                for (int u = 0; u < P; u++)
                    *reinterpret_cast<__half2 *>(row + dim(2 * u, lane)) =
                        __floats2half2_rn(clamp_to(x[j][2 * u], 65504.f), clamp_to(x[j][2 * u + 1], 65504.f));
            }
        } else {
            float amax = 0.f;
#pragma unroll
            for (int j = 0; j < N; j++)
#pragma unroll
                for (int e = 0; e < 2 * P; e++) amax = fmaxf(amax, fabsf(x[j][e])); // rows past cnt are zeros, a NaN does not count
            amax = fminf(kq_warp_max(amax), 57344.f);
            // 448 = 1.75 * 2^8: the exponent of amax / 448, rounded up
            int ex = ((int)((__float_as_uint(amax) + 0x1FFFFFu) >> 23)) - 127 - 8;
            ex = min(max(ex, -15), 7);
            float s = __uint_as_float((uint32_t)(ex + 127) << 23);
            if (off > 0) {
                const float old = *scale;
                if (old < s) { // the rows that the block holds, under the new scale
                    const float ratio = old / s;
                    for (int i = lane; i < off * HD / 4; i += 32) {
                        uint32_t *w = reinterpret_cast<uint32_t *>(page) + i;
                        const uint32_t c = *w;
                        const uint32_t h0 = kq_e4m3x2_h2((uint16_t)c), h1 = kq_e4m3x2_h2((uint16_t)(c >> 16));
                        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&h0)), b = __half22float2(*reinterpret_cast<const __half2 *>(&h1));
                        *w = (uint32_t)kq_e4m3x2(a.x * ratio, a.y * ratio) | ((uint32_t)kq_e4m3x2(b.x * ratio, b.y * ratio) << 16);
                    }
                } else if (old >= s) {
                    s = fminf(old, 128.f);
                }
            }
            __syncwarp(); // every lane has read the old scale
            if (lane == 0) *scale = s;
            const float inv = 1.f / s;
#pragma unroll
            for (int j = 0; j < N; j++) {
                if (j >= cnt) continue;
                uint8_t *row = page + (off + j) * HD;
                uint16_t c[P];
#pragma unroll
                for (int u = 0; u < P; u++) c[u] = kq_e4m3x2(x[j][2 * u] * inv, x[j][2 * u + 1] * inv);
                if (HD == 64 && split) {
                    row[lane] = (uint8_t)c[0];
                    row[32 + lane] = (uint8_t)(c[0] >> 8);
                } else if (!split && P == 2) {
                    *reinterpret_cast<uint32_t *>(row + 4 * lane) = (uint32_t)c[0] | ((uint32_t)c[P - 1] << 16);
                } else {
#pragma unroll
                    for (int u = 0; u < P; u++) *reinterpret_cast<uint16_t *>(row + dim(2 * u, lane)) = c[u];
                }
            }
        }
    }
    // one head's new rows of the block; cs: cosines and sines of the rows' pairs
    __device__ static void run(const Rows &r, int64_t row, int kh, uint8_t *kp, uint8_t *vp, float *ks, float *vs, int off, int cnt, int lane,
                               const float2 (*cs)[HD / 2], bool on) {
        float x[N][2 * P];
        uint32_t nan = 0;
        load(x, r, r.v, row * r.v_stride + (int64_t)kh * HD, r.v_stride, cnt, lane);
#pragma unroll
        for (int j = 0; j < N; j++)
#pragma unroll
            for (int e = 0; e < 2 * P; e++)
                if (x[j][e] != x[j][e]) {
                    nan |= 1u << j;
                    x[j][e] = 0.f;
                }
        store(x, vp, vs, off, cnt, lane);
        load(x, r, r.k, row * r.k_stride + (int64_t)kh * HD, r.k_stride, cnt, lane);
#pragma unroll
        for (int j = 0; j < N; j++) {
            if (on && j < cnt) {
#pragma unroll
                for (int u = 0; u < P; u++) { // separately rounded products: the order of roundings of the plain formula
                    const int i0 = split ? (P == 2 ? u : 0) : 2 * u, i1 = split ? (P == 2 ? u + 2 : 1) : 2 * u + 1;
                    const int pair = split ? (P == 2 ? 2 * lane + u : lane) : P * lane + u;
                    const float2 t = cs[j][pair];
                    const float a = x[j][i0], b = x[j][i1];
                    x[j][i0] = __fsub_rn(__fmul_rn(a, t.x), __fmul_rn(b, t.y));
                    x[j][i1] = __fadd_rn(__fmul_rn(a, t.y), __fmul_rn(b, t.x));
                }
            }
            if (nan >> j & 1) x[j][0] = __uint_as_float(0x7FC00000u);
        }
        store(x, kp, ks, off, cnt, lane);
    }
};

// grid (groups of `group` rows, heads / WARPS).  A CTA takes the blocks whose first new row is in its group.
template <int HD, bool F8, bool SPLIT>
__global__ void __launch_bounds__(WARPS * 32) pages_append_kernel(KqPages c, KqBatch b, Rows r, int group, KqTurns turns) {
    KQ_PDL_ENTER();
    __shared__ float2 cs[KQ_PAGE_BLOCK][HD / 2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int r0 = blockIdx.x * group, r1 = min(b.rows, r0 + group);
    int row = r0;
    while (row < r1) { // CTA-uniform
        const int s = seq_of_row(b.row_start, b.n_seq, row, lane);
        if (s >= b.n_seq) return; // rows behind the last sequence
        const int2 own = kq_seq_rows(b, s);
        const int p0 = b.pos0[s];
        if (row < own.x || p0 < 0) { // rows before the first sequence; a sequence without positions
            const int next = row < own.x ? own.x : own.y;
            if (next <= row) return; // row_start does not ascend
            row = next;
            continue;
        }
        const int64_t pos = (int64_t)p0 + row - own.x;
        const int off = (int)(pos % KQ_PAGE_BLOCK), cnt = min(KQ_PAGE_BLOCK - off, own.y - row);
        if (cnt <= 0) return;
        const int pg = kq_page_of(c, s, pos);
        if ((row == own.x || off == 0) && pg >= 0) {
            __syncthreads(); // the table of the block before has been read
            if (turns.on)
                for (int i = threadIdx.x; i < cnt * (HD / 2); i += WARPS * 32) cs[i / (HD / 2)][i % (HD / 2)] = kq_turn(turns.f[i % (HD / 2)], (int)pos + i / (HD / 2));
            __syncthreads();
            const int kh = blockIdx.y * WARPS + warp, in_page = (int)(pos % c.page) - off;
            if (kh < c.n_kv) {
                const int64_t code = (int64_t)pg * c.page_bytes + ((int64_t)kh * c.page + in_page) * HD * (F8 ? 1 : 2);
                const int64_t sc = F8 ? ((int64_t)pg * c.n_kv + kh) * (c.page / KQ_PAGE_BLOCK) + in_page / KQ_PAGE_BLOCK : 0;
                if (cnt == 1)
                    Block<HD, F8, 1, SPLIT>::run(r, row, kh, c.k + code, c.v + code, c.ks + sc, c.vs + sc, off, cnt, lane, cs, turns.on);
                else
                    Block<HD, F8, KQ_PAGE_BLOCK, SPLIT>::run(r, row, kh, c.k + code, c.v + code, c.ks + sc, c.vs + sc, off, cnt, lane, cs, turns.on);
            }
        }
        row += cnt;
    }
}

} // namespace

KqTurns kq_turns(float theta, int neox, int hd) {
    KqTurns t;
    t.on = theta > 0.f;
    t.neox = neox != 0;
    const double ratio = t.on ? pow((double)theta, -2.0 / hd) : 0.0; // one power: 63 products are off by 10^-14
    double f = t.on ? 1.0 / 6.283185307179586476925 : 0.0;
    for (int i = 0; i < 64; i++, f *= ratio) t.f[i] = i < hd / 2 ? (uint64_t)(f * 18446744073709551616.0) : 0;
    return t;
}

b200_status kq_pages_check(const char *who, const b200_kv_pages *c, const b200_page_batch *b, KqPages *out, KqBatch *batch) {
    KQ_REQUIRE(c && b, "%s: cache and batch required", who);
    const bool f8 = c->type == B200_TYPE_F8_E4M3;
    KQ_REQUIRE(f8 || c->type == B200_TYPE_F16, "%s: pages of type %u (f16 or e4m3)", who, c->type);
    KQ_REQUIRE(c->head_dim == 64 || c->head_dim == 128, "%s: head_dim %d (64 or 128)", who, c->head_dim);
    KQ_REQUIRE(c->page_size >= KQ_PAGE_BLOCK && c->page_size <= 4096 && c->page_size % KQ_PAGE_BLOCK == 0, "%s: pages of %d positions (a multiple of 16, up to 4096)", who, c->page_size);
    KQ_REQUIRE(c->n_kv >= 1 && c->n_kv <= 1024, "%s: %d KV heads", who, c->n_kv);
    KQ_REQUIRE(c->n_pages >= 1 && c->n_pages <= 0x7fffffff, "%s: %lld pages", who, (long long)c->n_pages);
    KQ_REQUIRE(c->k && c->v && ((((uintptr_t)c->k | (uintptr_t)c->v)) & 15) == 0, "%s: page pools must be given and 16-byte aligned", who);
    KQ_REQUIRE(!f8 || (c->k_scale && c->v_scale && (((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) & 3) == 0), "%s: e4m3 pages need their scales", who);
    const int64_t page = (int64_t)c->n_kv * c->page_size * c->head_dim, es = f8 ? 1 : 2, stride = c->page_stride ? c->page_stride : page;
    KQ_REQUIRE(stride >= page && stride * es % 16 == 0 && stride <= ((int64_t)1 << 36), "%s: page stride %lld (at least a page of %lld elements, a multiple of 16 bytes)", who, (long long)stride,
               (long long)page);
    KQ_REQUIRE(b->n_seq >= 0 && b->rows >= 0 && b->rows <= 0x3fffffff, "%s: %d sequences, %lld rows", who, b->n_seq, (long long)b->rows);
    KQ_REQUIRE(b->n_seq == 0 || (b->row_start && b->pos0 && b->table), "%s: row starts, positions and page table required", who);
    KQ_REQUIRE(((((uintptr_t)b->row_start | (uintptr_t)b->pos0 | (uintptr_t)b->table)) & 3) == 0, "%s: row starts, positions and page table must be 4-byte aligned", who);
    KQ_REQUIRE(b->table_len >= 0 && b->table_stride >= b->table_len, "%s: page table of %d entries, %d apart", who, b->table_len, b->table_stride);
    KQ_REQUIRE((int64_t)b->table_len * c->page_size <= 0x7fffffff, "%s: %d pages of %d positions are more than 2^31 - 1 positions", who, b->table_len, c->page_size);
    *out = KqPages{(uint8_t *)c->k, (uint8_t *)c->v, c->k_scale, c->v_scale, b->table, c->n_pages, stride * es, b->table_len, b->table_stride, c->page_size, c->n_kv};
    *batch = KqBatch{b->row_start, b->pos0, (int32_t)b->rows, b->n_seq};
    return B200_OK;
}

b200_status kq_rows_check(const char *who, const char *what, const void *p, uint32_t type, int64_t stride, int64_t width) {
    KQ_REQUIRE(type == B200_TYPE_F32 || type == B200_TYPE_F16 || type == B200_TYPE_BF16, "%s: %s of type %u (f32, f16 or bf16)", who, what, type);
    const int64_t es = type == B200_TYPE_F32 ? 4 : 2;
    KQ_REQUIRE(p && ((uintptr_t)p & 15) == 0 && stride >= width && stride * es % 16 == 0, "%s: %s must be 16-byte aligned rows, %lld elements or more apart", who, what, (long long)width);
    return B200_OK;
}

extern "C" b200_status b200_kv_pages_append(const b200_kv_pages *cache, const b200_page_batch *batch, uint32_t type, const void *k, int64_t k_stride,
                                            const void *v, int64_t v_stride, float theta, int32_t neox, void *stream) {
    KqPages c;
    KqBatch b;
    KQ_TRY(kq_pages_check("kv_pages_append", cache, batch, &c, &b));
    KQ_REQUIRE(theta >= 0.f && isfinite(theta), "kv_pages_append: rotation base %g", theta);
    if (b.rows == 0 || b.n_seq == 0) return B200_OK;
    const int64_t width = (int64_t)c.n_kv * cache->head_dim;
    KQ_TRY(kq_rows_check("kv_pages_append", "keys", k, type, k_stride, width));
    KQ_TRY(kq_rows_check("kv_pages_append", "values", v, type, v_stride, width));
    const Rows r{k, v, k_stride, v_stride, type};
    // few rows per sequence: a CTA per row, those of a sequence's later rows in a block have nothing to do; many: a CTA per 16 rows
    const int group = b.rows < 16 * (int64_t)b.n_seq ? 1 : KQ_PAGE_BLOCK;
    const dim3 grid((unsigned)kq_div_up(b.rows, group), (unsigned)kq_div_up(c.n_kv, WARPS));
    const KqTurns turns = kq_turns(theta, neox, cache->head_dim);
    const bool f8 = cache->type == B200_TYPE_F8_E4M3;
    const bool split = turns.on && turns.neox;
    auto *kern = cache->head_dim == 128 ? (f8 ? (split ? pages_append_kernel<128, true, true> : pages_append_kernel<128, true, false>)
                                              : (split ? pages_append_kernel<128, false, true> : pages_append_kernel<128, false, false>))
                                        : (f8 ? (split ? pages_append_kernel<64, true, true> : pages_append_kernel<64, true, false>)
                                              : (split ? pages_append_kernel<64, false, true> : pages_append_kernel<64, false, false>));
    kq_launch(kern, grid, WARPS * 32, 0, (cudaStream_t)stream, c, b, r, group, turns);
    KQ_COUNT_LAUNCH();
    KQ_LAUNCH_CHECK();
    return B200_OK;
}
