// How the kernels of b200_attention_pages share a ragged batch: the lengths are on the device, so every CTA works its part out itself.
//
// An item is one tile of R rows (row i of a sequence and KV head: new token i / G, query head i % G) of one sequence and KV head; its keys
// are cut into units of U positions.  All units of all items in order (sequence, head, tile, key) are cut into equal runs, one per CTA, so that
// the longest sequence does not decide how long the launch takes.  What an item costs besides its keys (queries in, rows out) counts as kq_setup
// units in front of its own; a CTA whose run ends among those leaves the item to the next.
//
// A CTA's run is at most the end of one item (its partial result goes into slot 2 cta), whole items (results go out), and the beginning of another
// (slot 2 cta + 1); meta[cta] describes the item that begins there and goes on in other CTAs, and a second kernel joins its slots in order.
// Nothing depends on timing.
#pragma once
#include "kq_pages.cuh"

struct KqAttnArgs {
    KqPages c;
    KqBatch b;
    const void *q;
    void *out;
    int64_t q_stride, out_stride;
    uint32_t type;
    int32_t G, window;
    int64_t t_lo, t_hi; // sequences with t_lo <= rows x G <= t_hi are this kernel's
    float scale_log2;
    KqTurns turns;
    float *part; // [2 CTAs][R (HD + 2)]: a slot is R unnormalised rows, then (maximum, sum) of each
    int4 *meta;  // [CTAs][2]: pieces (0: none), KV head, tile, -; first row and number of rows of the sequence, -, -
};

#ifdef __CUDACC__
struct KqSeq {
    int t, p0, row0;
    __device__ __forceinline__ int pos(int tok) const { return (int)min((int64_t)p0 + tok, (int64_t)0x7fffffff); }
};
__device__ __forceinline__ KqSeq kq_seq(const KqAttnArgs &a, int s) {
    const int2 r = kq_seq_rows(a.b, s);
    const int64_t n = (int64_t)(r.y - r.x) * a.G;
    return KqSeq{n >= a.t_lo && n <= a.t_hi ? r.y - r.x : 0, a.b.pos0[s], r.x};
}
template <int R> __device__ __forceinline__ int kq_tiles(const KqAttnArgs &a, int t) { return (t * a.G + R - 1) / R; }
// positions [x, y) that some row of the tile sees, x rounded down to a block, or for tiles of 256 rows to a whole unit
template <int R> __device__ __forceinline__ int2 kq_tile_keys(const KqAttnArgs &a, const KqSeq &q, int tile) {
    constexpr int A = R >= 128 ? 128 : KQ_PAGE_BLOCK;
    const int first = tile * R / a.G, last = min(q.t - 1, (tile * R + R - 1) / a.G); // rows x heads stay below 2^30
    const int64_t cap = (int64_t)a.c.table_len * a.c.page;
    const int hi = q.p0 < 0 ? 0 : (int)min((int64_t)q.p0 + last + 1, cap);
    const int lo = a.window > 0 ? (int)min(max((int64_t)0, (int64_t)q.p0 + first - a.window + 1), cap) & ~(A - 1) : 0;
    return make_int2(min(lo, hi & ~(A - 1)), hi);
}
// Units that setting an item up counts as.  200 decode sequences of 60 to 6000 positions: 188 us without any, 114 with two.  Prompts of 512 rows at
// 1536, f32 and bf16: 78 and 60 us with four, 78 and 57 with six, 82 and 56 with eight, 84 and 57 with ten.
template <int R> constexpr int kq_setup = R >= 128 ? 6 : 2;
template <int U> __device__ __forceinline__ int kq_units(int2 keys) { return max(1, (keys.y - keys.x + U - 1) / U); }
// units of one KV head of a sequence; the tiles' last tokens are counted on, not divided out
template <int R, int U> __device__ __forceinline__ long long kq_head_units(const KqAttnArgs &a, const KqSeq &q) {
    const int tiles = kq_tiles<R>(a, q.t);
    if (tiles <= 1 || a.window > 0) {
        long long n = 0;
        for (int i = 0; i < tiles; i++) n += kq_units<U>(kq_tile_keys<R>(a, q, i)) + kq_setup<R>;
        return n;
    }
    if (q.p0 < 0) return (long long)tiles * (1 + kq_setup<R>);
    long long n = 0;
    const int cap = a.c.table_len * a.c.page, room = cap - q.p0; // new tokens that have a place; below 2^31 by the checks
    const int dq = R / a.G, dr = R % a.G;
    int last = (R - 1) / a.G, rem = (R - 1) % a.G;
#pragma unroll 4
    for (int i = 0; i < tiles; i++) {
        const int seen = min(min(last, q.t - 1) + 1, room);
        n += ((uint32_t)max(q.p0 + seen, 1) + U - 1u) / U + kq_setup<R>;
        last += dq;
        rem += dr;
        if (rem >= a.G) {
            rem -= a.G;
            last++;
        }
    }
    return n;
}

// counts fit 32 bits but for absurd batches
__device__ __forceinline__ long long kq_div(long long a, long long b) { return ((a | b) >> 31) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b; }

// this CTA's run of units: [u0, u1), beginning `off` units into sequence s
struct KqRun {
    long long u0, u1, off, per_head; // per_head: units of a KV head of s
    int s;
};
template <int R, int U, int NT> __device__ KqRun kq_find_run(const KqAttnArgs &a) {
    __shared__ long long warp_sum[NT / 32], s_off, s_head;
    __shared__ int s_seq;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int each = (a.b.n_seq + NT - 1) / NT, i0 = min(a.b.n_seq, tid * each), i1 = min(a.b.n_seq, i0 + each);
    long long sum = 0, head = 0;
    for (int i = i0; i < i1; i++) {
        head = kq_head_units<R, U>(a, kq_seq(a, i));
        sum += head * a.c.n_kv;
    }
    long long inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
    }
    if (lane == 31) warp_sum[warp] = inc;
    if (tid == 0) s_seq = a.b.n_seq;
    __syncthreads();
    long long before = inc - sum, total = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; w++) {
        if (w < warp) before += warp_sum[w];
        total += warp_sum[w];
    }
    const long long per = max(1ll, kq_div(total + gridDim.x - 1, gridDim.x)), u0 = per * blockIdx.x;
    if (u0 >= before && u0 < before + sum) {
        long long off = u0 - before;
        for (int i = i0; i < i1; i++) {
            const long long h = i1 - i0 == 1 ? head : kq_head_units<R, U>(a, kq_seq(a, i)), n = h * a.c.n_kv;
            if (off < n) {
                s_seq = i;
                s_off = off;
                s_head = h;
                break;
            }
            off -= n;
        }
    }
    __syncthreads();
    KqRun r{u0, min(total, u0 + per), 0, 1, s_seq};
    if (r.s < a.b.n_seq) {
        r.off = s_off;
        r.per_head = s_head;
    } else r.u1 = r.u0;
    return r;
}
#endif

// sequences of few rows (any number is right), and its workspace
size_t kq_pages_decode_scratch(int hd);
b200_status kq_pages_decode(KqAttnArgs a, bool f8, int hd, int64_t most, uint8_t *scratch, cudaStream_t st);
// sequences of many rows
size_t kq_pages_prompt_scratch(int hd);
b200_status kq_pages_prompt(KqAttnArgs a, bool f8, int hd, uint8_t *scratch, cudaStream_t st);
