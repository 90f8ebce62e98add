// New keys and values into the pages of their sequences, the keys rotated on the way (b200_kv_pages_append).
//
// One CTA takes the new rows that fall into one aligned block of 16 positions of one sequence and 4 or 8 heads: 16-byte asynchronous copies
// bring them into shared memory while the CTA works out their cosines and sines, a lane turns and rounds the same pair of dimensions of every row of a
// head, and the rows go out from shared memory again as whole runs of their page (from the lanes, where a pair is (i, i + hd / 2), they went out
// a byte at a time: 11516 rows of 8 heads, bf16 into e4m3, 66 us against 38 with neighbouring pairs).  An e4m3 block is one CTA's own, so its
// scale (the smallest power of two that brings the largest of the new values to at most 448, never less than the scale of rows the block
// holds already) needs no atomics and does not depend on timing; rows it holds are rescaled in place when the scale grows.
//
// Bound by issue slots where rows are many (0.74 of them; 11516 rows of 8 heads, bf16: 30 us into e4m3 and into f16, where the bytes take 11 and 14), by
// one chain of dependent loads (whose row, which page, the row) where they are few (2.9 us a row in a captured graph).
//
// What no attention may meet behind a mask stays out of the values: a value beyond the page type's range goes in as the largest
// one (f16 65504, e4m3 448 * 2^7), and a NaN in v goes in as 0 with a NaN at its place in the token's k, so that every query that
// sees the token gets NaN and no other does.
#include "kq_pages.cuh"

#include <math.h>

#include <algorithm>
#include <type_traits>

namespace {

constexpr int WH = 2; // warps of a head: each takes every second row

struct Rows {
    const void *k, *v;
    int64_t k_stride, v_stride;
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

__device__ __forceinline__ float clamped(float x, float m) { // NaN stays
    x = x > m ? m : x;
    return x < -m ? -m : x;
}

template <int HD, bool F8, typename T, int H> struct Room { // shared memory: rows as they come, [keys, values][row][head][HD], and as they are stored, [keys, values][head][row][ROW]
    static constexpr int HEADS = H, WARPS = WH * H, ROW = HD * (F8 ? 1 : 2);
    static constexpr int IN = KQ_PAGE_BLOCK * HEADS * HD * (int)sizeof(T), OUT = HEADS * KQ_PAGE_BLOCK * ROW, SMEM = 2 * (IN + OUT);
};

// The new rows of one block from `in` to `out`.  A lane has P = HD / 64 neighbouring pairs of dimensions of a row, P lane ...: (pair, pair + HD / 2) if SPLIT,
// else (2 pair, 2 pair + 1).  For an e4m3 block the rows are turned twice, for the largest value and again for the codes: kept in registers they would
// halve the CTAs on an SM.
template <int HD, bool F8, typename T, bool SPLIT, int H>
__device__ __forceinline__ void convert(const uint8_t *in, uint8_t *out, bool mine, uint8_t *kp, uint8_t *vp, float *ks, float *vs, float old_k, float old_v, int off, int cnt,
                                        const float2 (*cs)[HD / 2], float (*top)[WH * H], bool on) {
    using M = Room<HD, F8, T, H>;
    constexpr int HEADS = H;
    constexpr int P = HD / 64;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % WH, head = warp / WH;
    // elements of a row as they stand: 2 P of them from d0 on, or P from d0 and P from d0 + HD / 2
    const int d0 = (SPLIT ? P : 2 * P) * lane;
    auto load = [&](const uint8_t *at, int j, float (&x)[2 * P]) {
        const T *row = reinterpret_cast<const T *>(at) + (j * HEADS + head) * HD + d0;
        if constexpr (P == 2) {
            const float2 a = kq_ld2(row), b = kq_ld2(row + (SPLIT ? HD / 2 : 2));
            x[0] = a.x, x[1] = a.y, x[2 * P - 2] = b.x, x[2 * P - 1] = b.y;
        } else if constexpr (SPLIT) x[0] = (float)row[0], x[1] = (float)row[HD / 2];
        else {
            const float2 a = kq_ld2(row);
            x[0] = a.x, x[1] = a.y;
        }
    };
    auto pair = [&](int j, float (&k)[2 * P], float (&v)[2 * P]) {
        load(in, j, k);
        load(in + M::IN, j, v);
        if (on) {
#pragma unroll
            for (int u = 0; u < P; u++) { // separately rounded products: the order of roundings of the plain formula
                const int e0 = SPLIT ? u : 2 * u, e1 = SPLIT ? u + P : 2 * u + 1;
                const float2 t = cs[j][P * lane + u];
                const float a = k[e0], b = k[e1];
                k[e0] = __fsub_rn(__fmul_rn(a, t.x), __fmul_rn(b, t.y));
                k[e1] = __fadd_rn(__fmul_rn(a, t.y), __fmul_rn(b, t.x));
            }
        }
        bool nan = false;
#pragma unroll
        for (int e = 0; e < 2 * P; e++) nan = nan || v[e] != v[e];
        if (nan) {
#pragma unroll
            for (int e = 0; e < 2 * P; e++)
                if (v[e] != v[e]) v[e] = 0.f, k[e] = __uint_as_float(0x7FC00000u);
        }
    };
    float inv[2] = {1.f, 1.f};
    if constexpr (F8) {
        float kmax = 0.f, vmax = 0.f;
#pragma unroll 2
        for (int j = part; j < cnt; j += WH) {
            float k[2 * P], v[2 * P];
            pair(j, k, v);
#pragma unroll
            for (int e = 0; e < 2 * P; e++) kmax = fmaxf(kmax, fabsf(k[e])), vmax = fmaxf(vmax, fabsf(v[e])); // a NaN does not count
        }
        kmax = kq_warp_top(kmax);
        vmax = kq_warp_top(vmax);
        if (lane == 0) top[0][warp] = kmax, top[1][warp] = vmax;
        __syncthreads(); // every warp has also read the old scales
#pragma unroll
        for (int n = 0; n < 2; n++) {
            float amax = top[n][warp - part];
#pragma unroll
            for (int w = 1; w < WH; w++) amax = fmaxf(amax, top[n][warp - part + w]);
            amax = fminf(amax, 57344.f);
            // 448 = 1.75 * 2^8: the exponent of amax / 448, rounded up
            const int ex = min(max((int)((__float_as_uint(amax) + 0x1FFFFFu) >> 23) - 127 - 8, -15), 7);
            float s = __uint_as_float((uint32_t)(ex + 127) << 23);
            const float old = n ? old_v : old_k;
            if (off > 0 && mine) {
                if (old < s) { // the rows that the block holds, under the new scale
                    const float ratio = old / s;
                    for (int x = part * 32 + lane; x < off * HD / 4; x += 32 * WH) {
                        uint32_t *w = reinterpret_cast<uint32_t *>(n ? vp : kp) + x;
                        const uint32_t c = *w;
                        uint32_t h0, h1;
                        kq_e4m3x4_h2(c, h0, h1);
                        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&h0)), b = __half22float2(*reinterpret_cast<const __half2 *>(&h1));
                        *w = (uint32_t)kq_e4m3x2(a.x * ratio, a.y * ratio) | ((uint32_t)kq_e4m3x2(b.x * ratio, b.y * ratio) << 16);
                    }
                } else if (old >= s) {
                    s = fminf(old, 128.f);
                }
            }
            if (part == 0 && lane == 0 && mine) *(n ? vs : ks) = s;
            inv[n] = 1.f / s;
        }
    }
#pragma unroll 2
    for (int j = part; j < cnt; j += WH) {
        float x[2][2 * P];
        pair(j, x[0], x[1]);
#pragma unroll
        for (int n = 0; n < 2; n++) {
            uint8_t *row = out + n * M::OUT + (head * KQ_PAGE_BLOCK + j) * M::ROW;
            if constexpr (F8) {
                uint16_t c[P];
#pragma unroll
                for (int u = 0; u < P; u++) c[u] = kq_e4m3x2(x[n][2 * u] * inv[n], x[n][2 * u + 1] * inv[n]); // elements as they stand
                if constexpr (SPLIT && P == 1) row[d0] = (uint8_t)c[0], row[d0 + HD / 2] = (uint8_t)(c[0] >> 8);
                else if constexpr (SPLIT) *reinterpret_cast<uint16_t *>(row + d0) = c[0], *reinterpret_cast<uint16_t *>(row + d0 + HD / 2) = c[P - 1];
                else if constexpr (P == 1) *reinterpret_cast<uint16_t *>(row + d0) = c[0];
                else *reinterpret_cast<uint32_t *>(row + d0) = (uint32_t)c[0] | (uint32_t)c[P - 1] << 16;
            } else {
                __half2 c[P];
                __half *h = reinterpret_cast<__half *>(row);
#pragma unroll
                for (int u = 0; u < P; u++) c[u] = __floats2half2_rn(clamped(x[n][2 * u], 65504.f), clamped(x[n][2 * u + 1], 65504.f));
                if constexpr (SPLIT && P == 1) h[d0] = __low2half(c[0]), h[d0 + HD / 2] = __high2half(c[0]);
                else if constexpr (SPLIT) *reinterpret_cast<__half2 *>(h + d0) = c[0], *reinterpret_cast<__half2 *>(h + d0 + HD / 2) = c[P - 1];
                else {
#pragma unroll
                    for (int u = 0; u < P; u++) reinterpret_cast<__half2 *>(h + d0)[u] = c[u];
                }
            }
        }
    }
}

// grid (groups of `group` rows, heads in parts).  A CTA takes the blocks whose first new row is in its group.
template <int HD, bool F8, typename T, bool SPLIT, int H>
__global__ void __launch_bounds__(WH * H * 32, 16 / H) pages_append_kernel(const __grid_constant__ KqPages c, const __grid_constant__ KqBatch b, const __grid_constant__ Rows r, int group,
                                                                     const __grid_constant__ KqTurns turns) {
    using M = Room<HD, F8, T, H>;
    constexpr int HEADS = M::HEADS, WARPS = M::WARPS;
    extern __shared__ __align__(16) uint8_t room[];
    __shared__ float2 cs[KQ_PAGE_BLOCK][HD / 2];
    __shared__ uint64_t turns_s[HD / 2]; // a lane's own entry is no broadcast: not from the constant bank
    __shared__ float top[2][WARPS];
    constexpr int NT = WARPS * 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, h0 = blockIdx.y * HEADS, heads = min(HEADS, c.n_kv - h0), kh = h0 + warp / WH;
    if (tid < HD / 2) turns_s[tid] = turns.f[tid];
    KQ_PDL_ENTER();
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
        const bool first = row == own.x || off == 0; // of its block
        __syncthreads();                             // the block before is out of `room`
        if (first) {                                 // rows on their way in, whether their page is there or not
            constexpr int PER = HEADS * HD * (int)sizeof(T) / 16; // 16-byte chunks of a row's heads
            for (int x = tid; x < 2 * KQ_PAGE_BLOCK * PER; x += NT) {
                const int n = x / (KQ_PAGE_BLOCK * PER), j = x / PER % KQ_PAGE_BLOCK, ch = x % PER;
                if (j >= cnt) continue;
                const T *src = (const T *)(n ? r.v : r.k) + (int64_t)(row + j) * (n ? r.v_stride : r.k_stride) + (int64_t)h0 * HD;
                if (ch < heads * (HD * (int)sizeof(T) / 16))
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(room + n * M::IN + (j * PER + ch) * 16)),
                                 "l"(reinterpret_cast<const uint8_t *>(src) + ch * 16)
                                 : "memory");
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        const int pg = first ? kq_page_of(c, s, pos) : -1;
        if (first) {
            const int in_page = (int)(pos % c.page) - off, h = min(kh, c.n_kv - 1);
            const bool mine = pg >= 0 && kh < c.n_kv;
            const int64_t page = (int64_t)max(pg, 0) * c.page_bytes;
            const int64_t code = page + ((int64_t)h * c.page + in_page) * M::ROW;
            const int64_t sc = F8 ? ((int64_t)max(pg, 0) * c.n_kv + h) * (c.page / KQ_PAGE_BLOCK) + in_page / KQ_PAGE_BLOCK : 0;
            float old_k = 0.f, old_v = 0.f;
            if (F8 && mine && off > 0) old_k = c.ks[sc], old_v = c.vs[sc];
            if (turns.on)
                for (int i = tid; i < cnt * (HD / 2); i += NT) cs[i / (HD / 2)][i % (HD / 2)] = kq_turn(turns_s[i % (HD / 2)], (int)pos + i / (HD / 2));
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncthreads();
            uint8_t *out = room + 2 * M::IN;
            convert<HD, F8, T, SPLIT, H>(room, out, mine, c.k + code, c.v + code, c.ks + sc, c.vs + sc, old_k, old_v, off, cnt, cs, top, turns.on);
            __syncthreads();
            // a head's new rows are one run of its page
            constexpr int PER = KQ_PAGE_BLOCK * M::ROW / 16;
            if (pg >= 0)
                for (int x = tid; x < 2 * HEADS * PER; x += NT) {
                    const int n = x / (HEADS * PER), hh = x / PER % HEADS, ch = x % PER;
                    if (hh >= heads || ch >= cnt * (M::ROW / 16)) continue;
                    uint8_t *dst = (n ? c.v : c.k) + page + ((int64_t)(h0 + hh) * c.page + in_page + off) * M::ROW;
                    *reinterpret_cast<uint4 *>(dst + ch * 16) = *reinterpret_cast<const uint4 *>(out + n * M::OUT + hh * KQ_PAGE_BLOCK * M::ROW + ch * 16);
                }
        }
        row += cnt;
    }
}

template <int HD, bool F8, typename T, bool SPLIT, int H> b200_status launch(const KqPages &c, const KqBatch &b, const Rows &r, const KqTurns &turns, cudaStream_t st) {
    using M = Room<HD, F8, T, H>;
    static bool attr[64];
    int dev = 0;
    KQ_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !attr[dev]) {
        KQ_CUDA(cudaFuncSetAttribute(pages_append_kernel<HD, F8, T, SPLIT, H>, cudaFuncAttributeMaxDynamicSharedMemorySize, M::SMEM));
        if (dev >= 0 && dev < 64) attr[dev] = true;
    }
    // few rows per sequence: a CTA per row, those of a sequence's later rows in a block have nothing to do; many: a CTA per 16 rows, which takes their
    // blocks one after another (256 sequences of a row 12.5 us with the first, 40 with the second; 4000 rows of one sequence 35 and 16)
    const int group = b.rows < 16 * (int64_t)b.n_seq ? 1 : KQ_PAGE_BLOCK;
    const dim3 grid((unsigned)kq_div_up(b.rows, group), (unsigned)kq_div_up(c.n_kv, H));
    kq_launch(pages_append_kernel<HD, F8, T, SPLIT, H>, grid, M::WARPS * 32, M::SMEM, st, c, b, r, group, turns);
    KQ_COUNT_LAUNCH();
    KQ_LAUNCH_CHECK();
    return B200_OK;
}
// heads of a CTA: 4, or 8 where rows and codes of 8 take less than half an SM (16-bit rows into e4m3: 11516 rows of 8 heads 30 us instead of 32;
// into f16 36 instead of 30); they share their angles
template <int HD, bool F8, typename T> b200_status launch(const KqPages &c, const KqBatch &b, const Rows &r, const KqTurns &turns, cudaStream_t st) {
    const bool split = turns.on && turns.neox;
    if constexpr (F8 && sizeof(T) == 2)
        if (c.n_kv > 4) return split ? launch<HD, F8, T, true, 8>(c, b, r, turns, st) : launch<HD, F8, T, false, 8>(c, b, r, turns, st);
    return split ? launch<HD, F8, T, true, 4>(c, b, r, turns, st) : launch<HD, F8, T, false, 4>(c, b, r, turns, st);
}
template <int HD, bool F8> b200_status launch(uint32_t type, const KqPages &c, const KqBatch &b, const Rows &r, const KqTurns &turns, cudaStream_t st) {
    if (type == B200_TYPE_F32) return launch<HD, F8, float>(c, b, r, turns, st);
    return type == B200_TYPE_F16 ? launch<HD, F8, __half>(c, b, r, turns, st) : launch<HD, F8, __nv_bfloat16>(c, b, r, turns, st);
}

} // namespace

KqTurns kq_turns(float theta, int neox, int hd) {
    KqTurns t;
    t.on = theta > 0.f;
    t.neox = neox != 0;
    const double ratio = t.on ? pow((double)theta, -2.0 / hd) : 0.0; // one power: 63 products are off by 5.5e-15 at most (bases from 0.01 to 10^9)
    double f = t.on ? 1.0 / 6.283185307179586476925 : 0.0;
    for (int i = 0; i < 64; i++, f *= ratio) t.f[i] = i < hd / 2 ? (uint64_t)((f - floor(f)) * 18446744073709551616.0) : 0; // a base below 1 turns faster than once a position
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
    KQ_REQUIRE(stride >= page && stride * es % 16 == 0 && stride <= KQ_MOST_ELEMENTS / c->n_pages && stride <= ((int64_t)1 << 36), "%s: page stride %lld (at least a page of %lld elements, a multiple of 16 bytes)", who, (long long)stride,
               (long long)page);
    KQ_REQUIRE(b->n_seq >= 0 && b->rows >= 0 && b->rows <= 0x3fffffff, "%s: %d sequences, %lld rows", who, b->n_seq, (long long)b->rows);
    KQ_REQUIRE(b->n_seq == 0 || (b->row_start && b->pos0 && (b->table || b->table_len == 0)), "%s: row starts, positions and page table required", who);
    KQ_REQUIRE(((((uintptr_t)b->row_start | (uintptr_t)b->pos0 | (uintptr_t)b->table)) & 3) == 0, "%s: row starts, positions and page table must be 4-byte aligned", who);
    KQ_REQUIRE(b->table_len >= 0 && b->table_stride >= b->table_len, "%s: page table of %d entries, %d apart", who, b->table_len, b->table_stride);
    // the attention kernels' steps run up to 4095 positions past the last one
    KQ_REQUIRE((int64_t)b->table_len * c->page_size <= 0x7ffff000, "%s: %d pages of %d positions are more than 2^31 - 4096 positions", who, b->table_len, c->page_size);
    *out = KqPages{(uint8_t *)c->k, (uint8_t *)c->v, c->k_scale, c->v_scale, b->table, c->n_pages, stride * es, b->table_len, b->table_stride, c->page_size, c->n_kv};
    *batch = KqBatch{b->row_start, b->pos0, (int32_t)b->rows, b->n_seq};
    return B200_OK;
}

b200_status kq_rows_check(const char *who, const char *what, const void *p, uint32_t type, int64_t rows, int64_t stride, int64_t width) {
    KQ_REQUIRE(type == B200_TYPE_F32 || type == B200_TYPE_F16 || type == B200_TYPE_BF16, "%s: %s of type %u (f32, f16 or bf16)", who, what, type);
    const int64_t es = type == B200_TYPE_F32 ? 4 : 2;
    // products of rows and strides stay far from 64 bits
    KQ_REQUIRE(stride <= KQ_MOST_ELEMENTS / std::max<int64_t>(rows, 1), "%s: %s of %lld rows, %lld elements apart", who, what, (long long)rows, (long long)stride);
    KQ_REQUIRE(p && ((uintptr_t)p & 15) == 0 && stride >= width && stride * es % 16 == 0, "%s: %s must be 16-byte aligned rows, %lld elements or more apart", who, what, (long long)width);
    return B200_OK;
}

namespace {
int pool_spans(const b200_kv_pages *c, KqSpan *out) { // keys, values and, for e4m3, their scales
    const bool f8 = c->type == B200_TYPE_F8_E4M3;
    const int64_t page = (int64_t)c->n_kv * c->page_size * c->head_dim, scales = c->n_pages * c->n_kv * (c->page_size / KQ_PAGE_BLOCK) * (int64_t)sizeof(float);
    out[0] = kq_rows_span("the pool of keys", c->k, f8 ? 1 : 2, c->n_pages, c->page_stride ? c->page_stride : page, page);
    out[1] = kq_rows_span("the pool of values", c->v, f8 ? 1 : 2, c->n_pages, c->page_stride ? c->page_stride : page, page);
    if (!f8) return 2;
    out[2] = KqSpan("the scales of keys", c->k_scale, scales);
    out[3] = KqSpan("the scales of values", c->v_scale, scales);
    return 4;
}
// what append writes must not lie over one another; pages of keys and values may take turns in one allocation
b200_status pools_apart(const char *who, const b200_kv_pages *c) {
    KqSpan pool[4];
    const int n = pool_spans(c, pool);
    for (int i = 0; i < n; i++)
        for (int j = i + 1; j < n; j++) {
            if (!pool[i].over(pool[j])) continue;
            bool turns = false;
            if (j == 1 && c->page_stride) {
                const uintptr_t es = n == 4 ? 1 : 2, page = (uintptr_t)c->n_kv * c->page_size * c->head_dim * es, stride = (uintptr_t)c->page_stride * es;
                const uintptr_t apart = (pool[0].from < pool[1].from ? pool[1].from - pool[0].from : pool[0].from - pool[1].from) % stride;
                turns = apart >= page && apart + page <= stride;
            }
            KQ_REQUIRE(turns, "%s: %s over %s", who, pool[i].what, pool[j].what);
        }
    return B200_OK;
}
} // namespace

b200_status kq_pages_apart(const char *who, const b200_kv_pages *c, const KqSpan &x) {
    KqSpan pool[4];
    for (int i = 0, n = pool_spans(c, pool); i < n; i++) KQ_REQUIRE(!x.over(pool[i]), "%s: %s over %s", who, x.what, pool[i].what);
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
    KQ_TRY(kq_rows_check("kv_pages_append", "keys", k, type, b.rows, k_stride, width));
    KQ_TRY(kq_rows_check("kv_pages_append", "values", v, type, b.rows, v_stride, width));
    const int64_t es = type == B200_TYPE_F32 ? 4 : 2;
    KQ_TRY(pools_apart("kv_pages_append", cache));
    KQ_TRY(kq_pages_apart("kv_pages_append", cache, kq_rows_span("new keys", k, es, b.rows, k_stride, width)));
    KQ_TRY(kq_pages_apart("kv_pages_append", cache, kq_rows_span("new values", v, es, b.rows, v_stride, width)));
    const Rows r{k, v, k_stride, v_stride};
    const KqTurns turns = kq_turns(theta, neox, cache->head_dim);
    const bool f8 = cache->type == B200_TYPE_F8_E4M3;
    if (cache->head_dim == 128) return f8 ? launch<128, true>(type, c, b, r, turns, (cudaStream_t)stream) : launch<128, false>(type, c, b, r, turns, (cudaStream_t)stream);
    return f8 ? launch<64, true>(type, c, b, r, turns, (cudaStream_t)stream) : launch<64, false>(type, c, b, r, turns, (cudaStream_t)stream);
}
