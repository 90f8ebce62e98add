// Attention of a few new rows per sequence over paged keys and values (b200_attention_pages): decode steps and drafts.
//
// A warp takes 16 positions (f16) or 32 (e4m3) of an item at a time through its own ring in shared memory, filled by 16-byte
// asynchronous copies (what no row sees, or is not there, arrives as zeros), so that loads stay in flight under the arithmetic and no warp waits for another.
// From there the fragments of mma.m16n8k16 are 16-byte reads: the order of a product's inner index is free, so the 16 bytes that a thread reads of a
// key are the dimensions that its lane holds in consecutive steps of Q K^T, and Q is laid out to match; of the values it
// reads 16 bytes of four keys and pairs them up by byte permutes into the rows of V^T.  16-byte chunks are stored at chunk ^ (row % 8), which keeps both
// kinds of read off each other's banks.  e4m3 codes become f16 in registers (K's scale goes onto the score, V's onto the product, both
// exact powers of two).  Scores are Q K^T with the item's rows as the 16 rows of the tile; the probabilities are then already the
// B operand of O^T = V^T P^T.  Softmax in base 2, statistics in 32 bits.
// A query row enters divided by the power of two that brings its largest element to [1, 2), so f16 neither overflows nor loses small
// rows; f32 and f16 rows go in as two f16 parts (rotation makes an f16 query longer than f16), and so do their probabilities; the tensor cores
// cut their sums off instead of rounding them, so those of one step (16 or 32 keys) are added to the row in 32-bit registers.  bf16 over f16 pages, whose
// results have 8 bits, lets the tensor cores add up a warp's steps (131072 keys in one CTA, one of which outweighs the others: 1.08 half steps off).
//
// Bound by HBM: a position costs 2 hd codes per KV head and is read once.  Whole calls, joining launch included: f16 pages, 200 sequences of 60 to 6000
// positions of 8 KV heads 6.2 TB/s, 0.95 of a copy's rate, 64 sequences of 4 KV heads 5.2; e4m3 pages, half the bytes for as much arithmetic, 200 sequences: 4.3 TB/s,
// where the instruction streams around the conversions count as much.  The units of
// all items are shared out evenly (kq_pages_sched.cuh), the four warps of a CTA take neighbouring positions and join their rows through shared memory at an item's end.
#include "kq_pages_sched.cuh"

#include <math.h>

#include <algorithm>
#include <type_traits>

namespace {

constexpr int NT = 128, NW = NT / 32;
constexpr int MAX_CTAS_PER_SM = 3;

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void *src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
// zeros where `there` is false (nothing is read then)
__device__ __forceinline__ void copy16_if(uint32_t dst, const void *src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void *src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint32_t word(const uint4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int HD, bool F8, int HT> struct Shape {
    static constexpr int R = 8 * HT, ES = F8 ? 1 : 2, ROW = HD * ES, NG = F8 ? 2 : 1, KT = 16 * NG; // groups of 16 positions of a warp's step
    static constexpr int STEP = 2 * KT * ROW;                                                       // keys, then values
    static constexpr int NST = STEP == 8192 ? (HT == 1 ? 2 : 3) : 4; // ring stages of a warp
    static constexpr int CTAS = HT == 1 ? 3 : 2;                     // per SM (2 of 3 stages each: 64 sequences 79 us instead of 75, 200 in 8 bits 208 instead of 188)
    static constexpr int SMEM = NW * NST * STEP;
    static_assert(NST * STEP >= R * HD * 4, "a warp's rows fit into its ring");
};
// place of 16-byte chunk c of row r
template <int ROW> __device__ __forceinline__ int place(int r, int c) { return r * ROW + ((c ^ (ROW >= 128 ? r & 7 : (r >> 1) & 3)) << 4); }

__device__ __noinline__ float2 turn_out_of_line(uint64_t f, int pos) { return kq_turn(f, pos); }

// HT: tiles of 8 rows (1 or 2); T: the activations' type, all but bf16 (whose results have 8 bits) with queries and probabilities in two f16 parts
template <int HD, bool F8, int HT, typename T>
__global__ void __launch_bounds__(NT, Shape<HD, F8, HT>::CTAS) pages_decode_kernel(const __grid_constant__ KqAttnArgs a) {
    using S = Shape<HD, F8, HT>;
    constexpr bool SPLIT = !std::is_same<T, __nv_bfloat16>::value;
    constexpr int R = S::R, ROW = S::ROW, NG = S::NG, KT = S::KT, U = NW * KT, NST = S::NST;
    constexpr int KL = ROW / 64, VL = (ROW + 127) / 128; // 16-byte reads of a key and of a value
    constexpr int KS = HD / 16, MT = HD / 16;            // steps of Q K^T, tiles of 16 dimensions of O^T
    constexpr int QP = HD + 4;
    extern __shared__ __align__(128) uint8_t ring_s[];
    __shared__ __align__(16) float q_s[R][QP];
    __shared__ float c_s[R];
    __shared__ float sc_s[NW][NST][4];  // scales of the step's groups: keys, values
    __shared__ int have_s[NW][NST];     // which of them are there
    __shared__ float m_s[NW][R], l_s[NW][R];
    __shared__ uint64_t turns_s[HD / 2]; // a lane's own entry is no broadcast: not from the constant bank
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    if (tid < HD / 2) turns_s[tid] = a.turns.f[tid];
    uint8_t *ring = ring_s + warp * (NST * S::STEP);
    const uint32_t ring_u = smem_u32(ring);
    auto o_at = [&](int w) { return reinterpret_cast<float (*)[HD]>(ring_s + w * (NST * S::STEP)); }; // a warp's rows, once its ring is done
    KQ_PDL_ENTER();
    KqRun run = kq_find_run<R, U, NT>(a);
    int4 meta = make_int4(0, 0, 0, 0), meta2 = meta;
    long long u = run.u0;
    for (int s = run.s; u < run.u1 && s < a.b.n_seq; s++, run.off = 0) {
        const KqSeq sq = kq_seq(a, s);
        if (sq.t == 0) continue;
        const int tiles = kq_tiles<R>(a, sq.t);
        const long long per_head = run.off ? run.per_head : 1; // only the sequence that the run begins in begins inside
        int kh = (int)kq_div(run.off, per_head), tile = 0;
        long long uo = run.off - kh * per_head;
        while (tile < tiles) { // the tile that the run begins in
            const int n = kq_units<U>(kq_tile_keys<R>(a, sq, tile)) + kq_setup<R>;
            if (uo < n) break;
            uo -= n;
            tile++;
        }
        for (; kh < a.c.n_kv && u < run.u1; kh++, tile = 0)
            for (; tile < tiles && u < run.u1; tile++, uo = 0) {
                const int2 keys = kq_tile_keys<R>(a, sq, tile);
                const int n_units = kq_units<U>(keys), part = (int)min((long long)n_units + kq_setup<R> - uo, run.u1 - u);
                const int ub = max(0, (int)uo - kq_setup<R>), take = max(0, (int)uo + part - kq_setup<R>) - ub;
                u += part;
                if (take == 0) continue; // the next CTA's
                // the queries' loads, under way while the positions are asked for
                float x[R / NW][HD / 32];
                int qtok[R / NW];
#pragma unroll
                for (int y = 0; y < R / NW; y++) {
                    const int rr = tile * R + warp + NW * y, tok = rr / a.G, h = kh * a.G + rr - tok * a.G;
                    const bool ok = tok < sq.t;
                    qtok[y] = tok;
                    const T *row = (const T *)a.q + (int64_t)(sq.row0 + (ok ? tok : 0)) * a.q_stride + (int64_t)(ok ? h : 0) * HD;
#pragma unroll
                    for (int i = 0; i < HD / 64; i++) {
                        const int pr = lane + 32 * i;
                        x[y][2 * i] = ok ? kq_ld1(row + (a.turns.neox ? pr : 2 * pr)) : 0.f;
                        x[y][2 * i + 1] = ok ? kq_ld1(row + (a.turns.neox ? pr + HD / 2 : 2 * pr + 1)) : 0.f;
                    }
                }
                __syncthreads(); // the item before has been joined
                const int bpp = a.c.page / KQ_PAGE_BLOCK;
                const int64_t head_off = (int64_t)kh * a.c.page * ROW;
                const int see_all = sq.pos(tile * R / a.G); // positions up to here every row sees ...
                const int see_from = a.window > 0 ? sq.pos(min((tile * R + R - 1) / a.G, sq.t - 1)) - a.window + 1 : 0; // ... from here on
                const int first_seen = a.window > 0 ? max(0, see_all - a.window + 1) : 0;                               // before this one none does
                // ---- asks for the positions of step i
                int pg[NG], inb[NG]; // page and block in it of this lane's step of the next 32
                auto ask = [&](int i) {
                    if (i >= take) {
                        copies_commit();
                        return;
                    }
                    if ((i & 31) == 0) {
#pragma unroll
                        for (int n = 0; n < NG; n++) {
                            const int key = keys.x + (ub + i + lane) * U + warp * KT + 16 * n;
                            pg[n] = -1;
                            inb[n] = 0;
                            if (i + lane < take && key < keys.y) {
                                const int blk = key / KQ_PAGE_BLOCK, pi = blk / bpp;
                                inb[n] = blk - pi * bpp;
                                const int id = pi < a.c.table_len ? a.c.table[(int64_t)s * a.c.table_stride + pi] : -1;
                                pg[n] = id >= 0 && id < a.c.n_pages ? id : -1;
                            }
                        }
                    }
                    const int st = i % NST, key0 = keys.x + (ub + i) * U + warp * KT;
                    int have = 0;
#pragma unroll
                    for (int n = 0; n < NG; n++) {
                        const int p = __shfl_sync(0xffffffffu, pg[n], i & 31), ib = __shfl_sync(0xffffffffu, inb[n], i & 31);
                        const int64_t off = (int64_t)max(p, 0) * a.c.page_bytes + head_off + (int64_t)ib * (KQ_PAGE_BLOCK * ROW);
                        have |= (p >= 0) << n;
                        constexpr int CH = ROW / 16, PER = 16 * CH / 32; // chunks of a row; copies of a lane
                        const uint32_t dst = ring_u + st * S::STEP;
                        const uint8_t *src_k = a.c.k + off + lane * 16, *src_v = a.c.v + off + lane * 16; // a block is one run: copy j of a lane is 512 j on
                        const int kg = key0 + 16 * n;
                        if (p >= 0 && kg + 16 <= keys.y && kg >= first_seen) {
#pragma unroll
                            for (int j = 0; j < PER; j++) {
                                const int x = j * 32 + lane;
                                copy16(dst + place<ROW>(16 * n + x / CH, x % CH), src_k + 512 * j);
                                copy16(dst + KT * ROW + place<ROW>(16 * n + x / CH, x % CH), src_v + 512 * j);
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < PER; j++) {
                                const int x = j * 32 + lane, key = kg + x / CH;
                                const bool there = p >= 0 && key < keys.y && key >= first_seen; // what no row sees may hold anything: it must not meet a probability of 0
                                copy16_if(dst + place<ROW>(16 * n + x / CH, x % CH), src_k + 512 * j, there);
                                copy16_if(dst + KT * ROW + place<ROW>(16 * n + x / CH, x % CH), src_v + 512 * j, there);
                            }
                        }
                        if (F8 && p >= 0 && lane < 2)
                            copy4(smem_u32(&sc_s[warp][st][2 * lane + n]), (lane ? a.c.vs : a.c.ks) + ((int64_t)p * a.c.n_kv + kh) * bpp + ib);
                    }
                    if (lane == 0) have_s[warp][st] = have;
                    copies_commit();
                };
                for (int i = 0; i < NST - 1; i++) ask(i);
                // ---- the item's queries: rotated, normed, in shared memory
#pragma unroll
                for (int y = 0; y < R / NW; y++) {
                    const int r = warp + NW * y;
                    float amax = 0.f;
#pragma unroll
                    for (int i = 0; i < HD / 64; i++) {
                        const float v0 = x[y][2 * i], v1 = x[y][2 * i + 1];
                        if (a.turns.on) {
                            const float2 cs = turn_out_of_line(turns_s[lane + 32 * i], sq.pos(qtok[y]));
                            x[y][2 * i] = v0 * cs.x - v1 * cs.y;
                            x[y][2 * i + 1] = v0 * cs.y + v1 * cs.x;
                        }
                        amax = fmaxf(amax, fmaxf(fabsf(x[y][2 * i]), fabsf(x[y][2 * i + 1])));
                    }
                    amax = kq_warp_top(amax);
                    const uint32_t e = min(max(__float_as_uint(amax) >> 23, 1u), 252u);
                    const float f = amax > 0.f ? __uint_as_float((254u - e) << 23) : 1.f;
#pragma unroll
                    for (int i = 0; i < HD / 64; i++) {
                        const int pr = lane + 32 * i;
                        q_s[r][a.turns.neox ? pr : 2 * pr] = x[y][2 * i] * f;
                        q_s[r][a.turns.neox ? pr + HD / 2 : 2 * pr + 1] = x[y][2 * i + 1] * f;
                    }
                    if (lane == 0) c_s[r] = amax > 0.f ? a.scale_log2 * __uint_as_float(e << 23) : a.scale_log2;
                }
                __syncthreads();
                // Q as the A operand: rows g and g + 8 of the tile.  Up to 8 rows: the second parts take the other 8 places of the same product.
                uint32_t qh[KS][4], ql[SPLIT && HT == 2 ? KS : 1][4];
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    const int d = F8 ? 64 * (ks >> 2) + 16 * t4 + 4 * (ks & 3) : 32 * (ks >> 1) + 8 * t4 + 4 * (ks & 1);
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const float4 v = *reinterpret_cast<const float4 *>(&q_s[g + (HT == 2 ? 8 * h : 0)][d]);
                        const uint32_t x = kq_h2(v.x, v.y), y = kq_h2(v.z, v.w);
                        if (HT == 2 || h == 0) {
                            qh[ks][h] = x;
                            qh[ks][h + 2] = y;
                            if (SPLIT && HT == 2) {
                                ql[SPLIT && HT == 2 ? ks : 0][h] = kq_h2_low(v.x, v.y, x);
                                ql[SPLIT && HT == 2 ? ks : 0][h + 2] = kq_h2_low(v.z, v.w, y);
                            }
                        } else {
                            qh[ks][h] = SPLIT ? kq_h2_low(v.x, v.y, x) : 0u;
                            qh[ks][h + 2] = SPLIT ? kq_h2_low(v.z, v.w, y) : 0u;
                        }
                    }
                }
                float crow[HT], m[HT], l[HT], o[HT][MT][4];
                int lim[HT]; // last position that row g (+ 8) sees
#pragma unroll
                for (int h = 0; h < HT; h++) {
                    crow[h] = c_s[g + 8 * h];
                    const int tok = min((tile * R + g + 8 * h) / a.G, sq.t - 1);
                    lim[h] = sq.p0 < 0 ? -1 : sq.pos(tok);
                    m[h] = -INFINITY;
                    l[h] = 0.f;
#pragma unroll
                    for (int i = 0; i < MT; i++) o[h][i][0] = o[h][i][1] = o[h][i][2] = o[h][i][3] = 0.f;
                }
                for (int i = 0; i < take; i++) {
                    copies_wait<NST - 2>();
                    __syncwarp(); // every lane's copies of step i are in, and every lane is done with the stage that is filled next
                    ask(i + NST - 1);
                    const int key0 = keys.x + (ub + i) * U + warp * KT, st = i % NST;
                    if (key0 >= keys.y) continue; // warp-uniform
                    const uint8_t *kst = ring + st * S::STEP, *vst = kst + KT * ROW;
                    const int have = have_s[warp][st];
                    // ---- scores
                    float sc[NG][2][4];
#pragma unroll
                    for (int n = 0; n < NG; n++)
#pragma unroll
                        for (int nt = 0; nt < 2; nt++) {
                            float(&c)[4] = sc[n][nt];
                            c[0] = c[1] = c[2] = c[3] = 0.f;
#pragma unroll
                            for (int j = 0; j < KL; j++) {
                                const uint4 kr = *reinterpret_cast<const uint4 *>(kst + place<ROW>(16 * n + 8 * nt + g, 4 * j + t4));
#pragma unroll
                                for (int x = 0; x < KS / KL; x++) {
                                    const int ks = j * (KS / KL) + x;
                                    uint32_t b0, b1;
                                    if (F8) kq_e4m3x4_h2(word(kr, x), b0, b1);
                                    else b0 = word(kr, 2 * x), b1 = word(kr, 2 * x + 1);
                                    mma(c, qh[ks], b0, b1);
                                    if (SPLIT && HT == 2) mma(c, ql[SPLIT && HT == 2 ? ks : 0], b0, b1);
                                }
                            }
                            if (SPLIT && HT == 1) {
                                c[0] += c[2];
                                c[1] += c[3];
                            }
                        }
                    float mx[HT];
#pragma unroll
                    for (int h = 0; h < HT; h++) mx[h] = -INFINITY;
#pragma unroll
                    for (int n = 0; n < NG; n++) {
                        const int kg = key0 + 16 * n;
                        const bool all = (have >> n & 1) && kg + 15 <= see_all && kg >= see_from;
#pragma unroll
                        for (int h = 0; h < HT; h++) {
                            const float f = F8 ? crow[h] * sc_s[warp][st][n] : crow[h];
#pragma unroll
                            for (int nt = 0; nt < 2; nt++)
#pragma unroll
                                for (int j = 0; j < 2; j++) {
                                    float &x = sc[n][nt][2 * h + j];
                                    x *= f;
                                    if (!all) {
                                        const int key = kg + 8 * nt + 2 * t4 + j;
                                        if (!(have >> n & 1) || key > lim[h] || key >= keys.y || (a.window > 0 && key <= lim[h] - a.window)) x = -INFINITY;
                                    }
                                    mx[h] = fmaxf(mx[h], x);
                                }
                        }
                    }
                    // ---- softmax
                    float alpha[HT];
                    bool same = true;
                    uint32_t ph[NG][HT][2], pl[SPLIT ? NG : 1][HT][2];
#pragma unroll
                    for (int h = 0; h < HT; h++) {
                        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
                        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
                        const float mn = fmaxf(m[h], mx[h]), sub = mn == -INFINITY ? 0.f : mn - 14.f;
                        alpha[h] = mn == -INFINITY ? 0.f : kq_ex2(m[h] - mn); // nothing seen before: 2^-inf = 0
                        same = same && m[h] == mn;
                        m[h] = mn;
                        float sum = 0.f;
#pragma unroll
                        for (int n = 0; n < NG; n++)
#pragma unroll
                            for (int nt = 0; nt < 2; nt++) {
                                const float p0 = kq_ex2(sc[n][nt][2 * h] - sub), p1 = kq_ex2(sc[n][nt][2 * h + 1] - sub); // up to 2^14: small ones keep their bits in f16
                                sum += p0 + p1;
                                ph[n][h][nt] = kq_h2(p0, p1);
                                if (SPLIT) pl[SPLIT ? n : 0][h][nt] = kq_h2_low(p0, p1, ph[n][h][nt]);
                            }
                        l[h] = l[h] * alpha[h] + sum;
                    }
                    if (!__all_sync(0xffffffffu, same)) { // columns of O^T are rows 2 t4 and 2 t4 + 1: their factors sit in other lanes
#pragma unroll
                        for (int h = 0; h < HT; h++) {
                            const float a0 = __shfl_sync(0xffffffffu, alpha[h], 8 * t4), a1 = __shfl_sync(0xffffffffu, alpha[h], 8 * t4 + 4);
#pragma unroll
                            for (int i = 0; i < MT; i++) {
                                o[h][i][0] *= a0;
                                o[h][i][1] *= a1;
                                o[h][i][2] *= a0;
                                o[h][i][3] *= a1;
                            }
                        }
                    }
                    // ---- values
                    uint4 vr[NG][4][VL];
#pragma unroll
                    for (int n = 0; n < NG; n++)
#pragma unroll
                        for (int x = 0; x < 4; x++) {
                            const int r = 16 * n + 2 * t4 + (x & 1) + (x >> 1) * 8;
                            if constexpr (ROW < 128) {
                                const uint2 v = *reinterpret_cast<const uint2 *>(vst + place<ROW>(r, g >> 1) + 8 * (g & 1));
                                vr[n][x][0] = make_uint4(v.x, v.y, 0, 0);
                            } else {
#pragma unroll
                                for (int j = 0; j < VL; j++) vr[n][x][j] = *reinterpret_cast<const uint4 *>(vst + place<ROW>(r, 8 * j + g));
                            }
                        }
                    float vsc[NG]; // a group's scale goes onto its product, exactly
#pragma unroll
                    for (int n = 0; n < NG; n++) vsc[n] = F8 && (have >> n & 1) ? sc_s[warp][st][2 + n] : 0.f;
#pragma unroll
                    for (int i = 0; i < MT; i++) {
#pragma unroll
                        for (int n = 0; n < NG; n++) {
                            uint32_t va[4];
                            if (F8) { // two tiles per word of four dimensions
                                const uint32_t pick = i & 1 ? 0x7362u : 0x5140u;
                                const uint32_t x = __byte_perm(word(vr[n][0][0], i >> 1), word(vr[n][1][0], i >> 1), pick);
                                const uint32_t y = __byte_perm(word(vr[n][2][0], i >> 1), word(vr[n][3][0], i >> 1), pick);
                                kq_e4m3x4_h2(x, va[0], va[1]);
                                kq_e4m3x4_h2(y, va[2], va[3]);
                            } else {
                                const uint32_t w0 = word(vr[n][0][i >> 2], i & 3), w1 = word(vr[n][1][i >> 2], i & 3);
                                const uint32_t w2 = word(vr[n][2][i >> 2], i & 3), w3 = word(vr[n][3][i >> 2], i & 3);
                                va[0] = __byte_perm(w0, w1, 0x5410u);
                                va[1] = __byte_perm(w0, w1, 0x7632u);
                                va[2] = __byte_perm(w2, w3, 0x5410u);
                                va[3] = __byte_perm(w2, w3, 0x7632u);
                            }
#pragma unroll
                            for (int h = 0; h < HT; h++) {
                                if (!SPLIT && !F8) {
                                    mma(o[h][i], va, ph[n][h][0], ph[n][h][1]);
                                    continue;
                                }
                                float part[4] = {0.f, 0.f, 0.f, 0.f};
                                if (SPLIT) mma(part, va, pl[SPLIT ? n : 0][h][0], pl[SPLIT ? n : 0][h][1]);
                                mma(part, va, ph[n][h][0], ph[n][h][1]);
#pragma unroll
                                for (int x = 0; x < 4; x++) o[h][i][x] = F8 ? fmaf(part[x], vsc[n], o[h][i][x]) : o[h][i][x] + part[x];
                            }
                        }
                    }
                }
                copies_wait<0>();
                // ---- the four warps' rows, joined in warp order
                __syncwarp();
#pragma unroll
                for (int h = 0; h < HT; h++) {
                    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
                    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
                    if (t4 == 0) {
                        m_s[warp][g + 8 * h] = m[h];
                        l_s[warp][g + 8 * h] = l[h];
                    }
#pragma unroll
                    for (int i = 0; i < MT; i++) {
                        const int d = F8 ? (HD / 8) * g + 2 * i : 64 * (i >> 2) + 8 * g + 2 * (i & 3);
                        *reinterpret_cast<float2 *>(&o_at(warp)[8 * h + 2 * t4][d]) = make_float2(o[h][i][0], o[h][i][2]);
                        *reinterpret_cast<float2 *>(&o_at(warp)[8 * h + 2 * t4 + 1][d]) = make_float2(o[h][i][1], o[h][i][3]);
                    }
                }
                __syncthreads();
                const bool whole = ub == 0 && take == n_units;
                const int slot = 2 * blockIdx.x + (ub == 0 ? 1 : 0);
                float *po = a.part + (int64_t)slot * R * (HD + 2), *pml = po + R * HD;
                if (ub == 0 && !whole) {
                    const int per = (int)min((long long)0x7fffffff, run.u1 - run.u0); // a CTA whose item goes on has a full run
                    meta = make_int4(1 + (n_units - take + per - 1) / per, kh, tile, 0);
                    meta2 = make_int4(sq.row0, sq.t, 0, 0);
                }
                constexpr int TR = 16, PER = HD / TR; // threads of a row, dimensions of a thread
#pragma unroll 1
                for (int r = tid / TR; r < R; r += NT / TR) {
                    const int rr = tile * R + r, tok = rr / a.G, d0 = (tid % TR) * 4;
                    if (tok >= sq.t) continue;
                    float mm = m_s[0][r], ll = 0.f, v[PER];
#pragma unroll
                    for (int w = 1; w < NW; w++) mm = fmaxf(mm, m_s[w][r]);
                    const float sub = mm == -INFINITY ? 0.f : mm;
#pragma unroll
                    for (int k = 0; k < PER; k++) v[k] = 0.f;
#pragma unroll
                    for (int w = 0; w < NW; w++) {
                        const float f = kq_ex2(m_s[w][r] - sub);
                        ll += f * l_s[w][r];
#pragma unroll
                        for (int k = 0; k < PER; k += 4) { // dimensions d0 + 16 k ..
                            const float4 y = *reinterpret_cast<const float4 *>(&o_at(w)[r][d0 + 16 * k]);
                            v[k] += f * y.x, v[k + 1] += f * y.y, v[k + 2] += f * y.z, v[k + 3] += f * y.w;
                        }
                    }
                    if (whole) {
                        const float inv = ll == 0.f ? 0.f : 1.f / ll;
                        T *out = (T *)a.out + (int64_t)(sq.row0 + tok) * a.out_stride + (int64_t)(kh * a.G + rr - tok * a.G) * HD + d0;
#pragma unroll
                        for (int k = 0; k < PER; k += 4) {
                            if constexpr (sizeof(T) == 4) *reinterpret_cast<float4 *>(out + 16 * k) = make_float4(v[k] * inv, v[k + 1] * inv, v[k + 2] * inv, v[k + 3] * inv);
                            else if constexpr (SPLIT) *reinterpret_cast<uint2 *>(out + 16 * k) = make_uint2(kq_h2(v[k] * inv, v[k + 1] * inv), kq_h2(v[k + 2] * inv, v[k + 3] * inv));
                            else {
                                const __nv_bfloat162 b[2] = {__floats2bfloat162_rn(v[k] * inv, v[k + 1] * inv), __floats2bfloat162_rn(v[k + 2] * inv, v[k + 3] * inv)};
                                *reinterpret_cast<uint2 *>(out + 16 * k) = *reinterpret_cast<const uint2 *>(b);
                            }
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < PER; k += 4) *reinterpret_cast<float4 *>(po + r * HD + d0 + 16 * k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
                        if (d0 == 0) *reinterpret_cast<float2 *>(pml + 2 * r) = make_float2(mm, ll);
                    }
                }
            }
    }
    if (tid == 0) {
        a.meta[2 * blockIdx.x] = meta;
        a.meta[2 * blockIdx.x + 1] = meta2;
    }
}

// CTA b: the item of up to 16 rows that begins in CTA b of the attention kernel and goes on in the next pieces - 1 of them.  A row's pieces are
// shared out over 512 / 32 / R warps, whose lanes are the dimensions; eight pieces' loads are in flight together.
// A chain of latencies: 7 us of the 55 of one sequence at 131000 (eight items of some 50 pieces).
template <int HD, int R> __global__ void __launch_bounds__(512) pages_combine_kernel(const __grid_constant__ KqAttnArgs a) {
    constexpr int W = 16 / R, N = HD / 64; // warps of a row, pairs of dimensions of a lane
    __shared__ float2 o_s[16][HD / 2];
    __shared__ float2 ml_s[16];
    KQ_PDL_ENTER();
    const int4 meta = a.meta[2 * blockIdx.x], seq = a.meta[2 * blockIdx.x + 1];
    if (meta.x == 0) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = warp / W, part = warp % W;
    float m = -INFINITY, l = 0.f;
    float2 o[N];
#pragma unroll
    for (int u = 0; u < N; u++) o[u] = make_float2(0.f, 0.f);
    for (int i0 = part; i0 < meta.x; i0 += 8 * W) {
        float2 ml[8], v[8][N];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int i = i0 + j * W;
            ml[j] = make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int u = 0; u < N; u++) v[j][u] = make_float2(0.f, 0.f);
            if (i < meta.x) { // piece 0 is slot 2 b + 1, piece i slot 2 (b + i)
                const float *p = a.part + (int64_t)(2 * (blockIdx.x + i) + (i == 0 ? 1 : 0)) * (R * (HD + 2));
                ml[j] = *reinterpret_cast<const float2 *>(p + R * HD + 2 * r);
#pragma unroll
                for (int u = 0; u < N; u++) v[j][u] = *reinterpret_cast<const float2 *>(p + r * HD + 2 * (lane + 32 * u));
            }
        }
        float mn = m;
#pragma unroll
        for (int j = 0; j < 8; j++) mn = fmaxf(mn, ml[j].x);
        const float sub = mn == -INFINITY ? 0.f : mn, f0 = kq_ex2(m - sub);
        l *= f0;
#pragma unroll
        for (int u = 0; u < N; u++) o[u].x *= f0, o[u].y *= f0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float f = kq_ex2(ml[j].x - sub);
            l += f * ml[j].y;
#pragma unroll
            for (int u = 0; u < N; u++) o[u].x += f * v[j][u].x, o[u].y += f * v[j][u].y;
        }
        m = mn;
    }
    if (W > 1) { // the row's warps, in order
#pragma unroll
        for (int u = 0; u < N; u++) o_s[warp][lane + 32 * u] = o[u];
        if (lane == 0) ml_s[warp] = make_float2(m, l);
        __syncthreads();
        if (part) return;
        float mn = m;
#pragma unroll
        for (int w = 1; w < W; w++) mn = fmaxf(mn, ml_s[warp + w].x);
        const float sub = mn == -INFINITY ? 0.f : mn, f0 = kq_ex2(m - sub);
        l *= f0;
#pragma unroll
        for (int u = 0; u < N; u++) o[u].x *= f0, o[u].y *= f0;
#pragma unroll
        for (int w = 1; w < W; w++) {
            const float2 ml = ml_s[warp + w];
            const float f = kq_ex2(ml.x - sub);
            l += f * ml.y;
#pragma unroll
            for (int u = 0; u < N; u++) {
                const float2 v = o_s[warp + w][lane + 32 * u];
                o[u].x += f * v.x, o[u].y += f * v.y;
            }
        }
    }
    const int rr = meta.z * R + r, tok = rr / a.G;
    if (tok >= seq.y) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int u = 0; u < N; u++)
        kq_st2_type(a.type, a.out, (int64_t)(seq.x + tok) * a.out_stride + (int64_t)(meta.y * a.G + rr - tok * a.G) * HD + 2 * (lane + 32 * u), o[u].x * inv, o[u].y * inv);
}

b200_status combine(const KqAttnArgs &a, int hd, int R, int ctas, cudaStream_t st) {
    kq_launch(hd == 128 ? (R == 8 ? pages_combine_kernel<128, 8> : pages_combine_kernel<128, 16>) : (R == 8 ? pages_combine_kernel<64, 8> : pages_combine_kernel<64, 16>), ctas, 512,
              0, st, a);
    KQ_COUNT_LAUNCH();
    KQ_LAUNCH_CHECK();
    return B200_OK;
}

template <int HD, bool F8, int HT, typename T> b200_status launch(const KqAttnArgs &a, cudaStream_t st, int *ctas) {
    using S = Shape<HD, F8, HT>;
    static bool attr[64];
    int dev = 0;
    KQ_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !attr[dev]) {
        KQ_CUDA(cudaFuncSetAttribute(pages_decode_kernel<HD, F8, HT, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
        if (dev >= 0 && dev < 64) attr[dev] = true;
    }
    *ctas = kq_sm_count() * S::CTAS;
    kq_launch(pages_decode_kernel<HD, F8, HT, T>, *ctas, NT, S::SMEM, st, a);
    KQ_COUNT_LAUNCH();
    KQ_LAUNCH_CHECK();
    return B200_OK;
}
template <int HD, bool F8, int HT> b200_status launch(const KqAttnArgs &a, cudaStream_t st, int *ctas) {
    if (a.type == B200_TYPE_F32) return launch<HD, F8, HT, float>(a, st, ctas);
    return a.type == B200_TYPE_F16 ? launch<HD, F8, HT, __half>(a, st, ctas) : launch<HD, F8, HT, __nv_bfloat16>(a, st, ctas);
}
template <int HD> b200_status launch(const KqAttnArgs &a, bool f8, int ht, cudaStream_t st) {
    int ctas = 0;
    if (f8) KQ_TRY(ht == 1 ? (launch<HD, true, 1>(a, st, &ctas)) : (launch<HD, true, 2>(a, st, &ctas)));
    else KQ_TRY(ht == 1 ? (launch<HD, false, 1>(a, st, &ctas)) : (launch<HD, false, 2>(a, st, &ctas)));
    return combine(a, HD, 8 * ht, ctas, st);
}

// Sequences of up to FEW rows of a KV head go to the kernel above, longer ones to the one for prompts, where the caller says there are any.
// Measured, 16 sequences at 3000 of 4 KV heads, f16 pages, f32, here and there: 16 rows 34 and 88 us, 48 rows 65 and 90, 96 rows 110 and 92.
constexpr int64_t FEW = 64;
bool prompts(int64_t G, int64_t max_rows) { return G * max_rows > FEW; }

constexpr size_t up256(size_t v) { return (v + 255) / 256 * 256; }

} // namespace

size_t kq_pages_decode_scratch(int hd) {
    const size_t ctas = (size_t)kq_sm_count() * MAX_CTAS_PER_SM;
    return up256(ctas * 2 * sizeof(int4)) + ctas * 2 * 16 * (hd + 2) * sizeof(float);
}

b200_status kq_pages_decode(KqAttnArgs a, bool f8, int hd, int64_t most, uint8_t *scratch, cudaStream_t st) {
    const int ht = most <= 8 ? 1 : 2;
    a.meta = (int4 *)scratch;
    a.part = (float *)(scratch + up256((size_t)kq_sm_count() * MAX_CTAS_PER_SM * 2 * sizeof(int4)));
    return hd == 128 ? launch<128>(a, f8, ht, st) : launch<64>(a, f8, ht, st);
}

extern "C" {

size_t b200_attention_pages_scratch_bytes(const b200_kv_pages *cache, int32_t n_head, int32_t max_rows) {
    if (!cache || (cache->head_dim != 64 && cache->head_dim != 128) || cache->n_kv < 1 || n_head < 1) return 0;
    const size_t few = kq_pages_decode_scratch(cache->head_dim);
    // the two kernels run one after the other: they share the room
    return prompts(n_head / cache->n_kv, max_rows) ? std::max(few, kq_pages_prompt_scratch(cache->head_dim)) : few;
}

b200_status b200_attention_pages(const b200_kv_pages *cache, const b200_page_batch *batch, uint32_t type, const void *q, int64_t q_stride, int32_t n_head,
                                 int32_t max_rows, float theta, int32_t neox, int32_t window, float scale, void *out, int64_t out_stride, void *scratch,
                                 size_t scratch_bytes, void *stream) {
    KqAttnArgs a = {};
    KQ_TRY(kq_pages_check("attention_pages", cache, batch, &a.c, &a.b));
    KQ_REQUIRE(n_head >= 1 && n_head <= 4096 && n_head % cache->n_kv == 0, "attention_pages: %d query heads on %d KV heads", n_head, cache->n_kv);
    KQ_REQUIRE(theta >= 0.f && isfinite(theta), "attention_pages: rotation base %g", theta);
    KQ_REQUIRE(scale >= 0.f && isfinite(scale), "attention_pages: scale %g", scale);
    KQ_REQUIRE(a.b.rows * (int64_t)n_head <= 0x3fffffff, "attention_pages: %d rows of %d heads", a.b.rows, n_head);
    KQ_REQUIRE(window >= 0 && window <= (1 << 30) && max_rows >= 0, "attention_pages: window %d, rows %d", window, max_rows);
    if (a.b.rows == 0 || a.b.n_seq == 0) return B200_OK;
    const int hd = cache->head_dim;
    KQ_TRY(kq_rows_check("attention_pages", "queries", q, type, a.b.rows, q_stride, (int64_t)n_head * hd));
    KQ_TRY(kq_rows_check("attention_pages", "results", out, type, a.b.rows, out_stride, (int64_t)n_head * hd));
    KQ_REQUIRE(scratch && ((uintptr_t)scratch & 15) == 0 && scratch_bytes >= b200_attention_pages_scratch_bytes(cache, n_head, max_rows),
               "attention_pages: scratch of %zu bytes, 16-byte aligned, required", b200_attention_pages_scratch_bytes(cache, n_head, max_rows));
    const int64_t es = type == B200_TYPE_F32 ? 4 : 2, width = (int64_t)n_head * hd * es, apart = (const uint8_t *)out - (const uint8_t *)q, row = q_stride * es;
    const int64_t in_row = ((apart % row) + row) % row; // where results begin in a row of queries, if both are parts of rows as long
    KQ_REQUIRE(apart >= (a.b.rows - 1) * row + width || -apart >= (a.b.rows - 1) * out_stride * es + width || (q_stride == out_stride && in_row >= width && in_row + width <= row),
               "attention_pages: results over queries");
    const KqSpan results = kq_rows_span("results", out, es, a.b.rows, out_stride, (int64_t)n_head * hd);
    const KqSpan room("scratch", scratch, b200_attention_pages_scratch_bytes(cache, n_head, max_rows));
    KQ_TRY(kq_pages_apart("attention_pages", cache, results));
    KQ_TRY(kq_pages_apart("attention_pages", cache, room));
    KQ_REQUIRE(!room.over(results) && !room.over(kq_rows_span("", q, es, a.b.rows, q_stride, (int64_t)n_head * hd)), "attention_pages: scratch over results or queries");
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.type = type;
    a.G = n_head / cache->n_kv;
    a.window = window;
    a.t_lo = 1;
    a.t_hi = INT64_MAX;
    a.scale_log2 = (scale > 0.f ? scale : 1.f / sqrtf((float)hd)) * 1.4426950408889634f;
    a.turns = kq_turns(theta, neox, hd);
    const bool f8 = cache->type == B200_TYPE_F8_E4M3, many = prompts(a.G, max_rows);
    if (many) a.t_hi = FEW;
    if (!many || a.b.n_seq > 1) KQ_TRY(kq_pages_decode(a, f8, hd, std::min<int64_t>(FEW, (int64_t)std::max(max_rows, 1) * a.G), (uint8_t *)scratch, (cudaStream_t)stream));
    if (!many) return B200_OK;
    a.t_lo = a.b.n_seq > 1 ? FEW + 1 : 1;
    a.t_hi = INT64_MAX;
    return kq_pages_prompt(a, f8, hd, (uint8_t *)scratch, (cudaStream_t)stream);
}

} // extern "C"
