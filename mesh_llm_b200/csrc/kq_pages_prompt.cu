// Attention of many new rows per sequence over paged keys and values (b200_attention_pages): prompts, on the 5th-generation tensor cores.
//
// A CTA works on two tiles of 128 rows (row i of a sequence and KV head: token i / G, head i % G) that share every tile of 128 keys: while
// the tensor cores multiply for one, the softmax warps of the other work.  S = Q K^T and O += P V are tcgen05.mma kind::f16 with S (columns
// 0 and 128) and O (256 and 384) in TMEM; a softmax thread owns a row: it writes its probabilities over scores that it has read, as f16, which
// are the A operand of the second product, and rescales its row of O only when its maximum has grown by more than 4 in base 2.  The first 64 keys'
// part of the second product runs under the exponentials of the others.  f32 queries go in as two f16 parts, and so do their probabilities; f16
// queries, which the rotation makes longer than f16, go in as two.  As in the kernel for few rows a query row is divided by the power of two of its
// largest element.
//
// K and V tiles go through a ring in the order K0 V0 K1 V1 ...; f16 pages arrive by tiled TMA, 64 dimensions x 16 .. 128 positions of a page
// to a box, with the 128-byte swizzle that both products read (V as an MN-major operand), pages that are not there as the zeros of an
// out-of-range coordinate; e4m3 pages arrive as raw rows by bulk copies and four warps turn them into the f16 tile of what they stand for.
//
// Bound, where items are long, by the tensor pipe (4 x 512 clocks for 256 rows x 128 keys at head_dim 128), the exponentials (16 a clock: 2 x 1024) and the
// issue slots, all three near 2000 of the 3300 clocks that a unit of bf16 takes; where they are short, by setting an item up (33 k clocks for a CTA's first, 27 k
// for another).  4096 rows of 40 heads behind 12288 positions, bf16: 0.97 PFLOP/s (1240 us, under the power cap); f32 2130 us, f16 1580.  Units are shared out evenly over one CTA per SM (kq_pages_sched.cuh).
// Every wait is bounded: on a time-out the kernel records an error, lets its copies land, frees its TMEM and returns.
#include "kq_pages_sched.cuh"
#include "kq_tc.cuh"

#include <math.h>
#include <string.h>

#include <type_traits>

namespace {

constexpr int R = 256, BK = 128, NSOFT = 256;
constexpr uint64_t LIMIT = 5 * KQ_WAIT_LIMIT_NS;
constexpr uint32_t COL_S = 0, COL_O = 256;
// f32: the tensor cores cut their sums off instead of rounding them: of a product what lies below 2^-25 of the sum that it joins, of a step's sum what lies
// below its 24 bits.  So O and the row's sum of probabilities are put aside and added up in 32 bits every FLUSH units, and as soon as a unit has added less than
// 1 / DOMINATED of what is there: what a unit of 128 keys loses is in proportion to what it joins, 1.9e-6 of that on average.  The sum is taken in O's
// steps and cut off as O is, first parts by adding so, second parts by CUT_HALF_BIT for a step where there are any of some weight: what O loses to its 24 bits
// cancels on average where it is divided by.  Relative error, 512 rows of 40 heads behind 3000 keys: values of either sign 1.1e-6; positive values 2.7e-6
// where keys weigh alike, at most 7.4e-6 where one outweighs the others (every six units alone 2.0e-5), less than 6e-7 where all weight is on one.  Five units
// instead of six: 1.0e-6 for 5 % of the time.
// Results of 16 bits put theirs aside for the same reason, when the loss nears an eighth of their half step (f16 32 units, bf16 128): without, 60000 keys cost
// an f16 result up to 5.0 half steps instead of 1.2, 150000 a bf16 result 2.1 instead of 1.03.
template <typename T> constexpr int FLUSH = std::is_same<T, float>::value ? 6 : std::is_same<T, __half>::value ? 32 : 128;
constexpr float CUT_HALF_BIT = 4.3e-8f; // half a last bit relative to the value, over mantissas of 1 to 2 as they come: 2^-24 / (2 ln 2)
constexpr float DOMINATED = 12.f;
// Probabilities are worked out under 2^(m - PEAK), m the row's maximum when it last moved, and m moves when it would grow by more than GROWTH: they
// stay below 2^(PEAK + GROWTH), and f16's smallest step of 2^-24 is 2^-35 of the largest.  (6 and 8: 60000 keys of e^-14 beside one of 1, 1.06e-5 off instead of 3.5e-6.)
constexpr float PEAK = 11.f, GROWTH = 4.f;

__device__ int g_pages_error;

constexpr int HALF = BK * 128; // 128 rows of 64 dimensions
// steps of a product, in the address field of a descriptor (16 bytes): 16 dimensions of a K-major operand (Q, K^T), 16 positions of V
__device__ __forceinline__ constexpr uint32_t step_k(int s) { return (s >> 2) * (HALF / 16) + (s & 3) * 2; }
__device__ __forceinline__ constexpr uint32_t step_mn(int s) { return s * (2048 / 16); }
__device__ __forceinline__ void arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void expect(uint32_t bar, uint32_t bytes) { asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t *r) { TMEM_LD32(taddr, r); }
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t *r) { TMEM_ST32(taddr, r); }
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t *r) { TMEM_ST16(taddr, r); }
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float add_f16(float c, uint32_t h) { // c and the lower f16 of h
    asm("add.rn.f32.f16 %0, %1, %2;" : "=f"(c) : "h"((uint16_t)h), "f"(c));
    return c;
}
// pairs of f32 in one register pair
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) { // NaN if one is
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ uint64_t exp2_sfu(uint64_t x) {
    const float2 v = unpack2(x);
    return pack2(kq_ex2(v.x), kq_ex2(v.y));
}
// 2^x = 2^n 2^f, n the nearest whole number (added into the exponent), |f| <= 1/2: the cubic of least largest relative error there,
// 7.5e-5 (a seventh of half a step of f16).  Below 2^-126 it gives next to nothing, as it should; a NaN is seen to with the maximum.
constexpr int POLY = 3;
__device__ __forceinline__ uint64_t exp2_poly(uint64_t x) {
    const float2 v = unpack2(x);
    x = pack2(fmaxf(v.x, -126.f), fmaxf(v.y, -126.f));
    const float magic = 12582912.f; // 1.5 * 2^23: adding it rounds to a whole number in the low bits
    const uint64_t t = add2(x, pack2(magic, magic)), f = fma2(add2(t, pack2(-magic, -magic)), pack2(-1.f, -1.f), x);
    uint64_t p = fma2(pack2(0.05517167f, 0.05517167f), f, pack2(0.24261114f, 0.24261114f));
    p = fma2(p, f, pack2(0.69326097f, 0.69326097f));
    p = fma2(p, f, pack2(0.99992806f, 0.99992806f));
    const float2 tt = unpack2(t), pp = unpack2(p);
    return pack2(__int_as_float(__float_as_int(pp.x) + (__float_as_int(tt.x) << 23)), __int_as_float(__float_as_int(pp.y) + (__float_as_int(tt.y) << 23)));
}

template <int HD, bool F8, int QS> struct Layout {
    static constexpr int TILE = BK * HD * 2, RAW = BK * HD;                     // an f16 tile of the ring, a raw e4m3 tile
    static constexpr int Q = 2 * QS * TILE;                                     // [part][tile of rows]
    static constexpr int NR = F8 ? (HD == 128 && QS == 2 ? 2 : 4) : 0;          // raw tiles
    static constexpr int FREE = 224 * 1024 - Q - NR * RAW, NS0 = FREE / TILE, NS = NS0 > 6 ? 6 : NS0; // ring slots
    static constexpr int RING = Q, RAWS = Q + NS * TILE, TOTAL = RAWS + NR * RAW + 1024;
    static_assert(NS >= 2, "the ring holds a tile of keys and one of values");
};
constexpr int MAX_SLOTS = 6;

struct Shared {
    uint64_t full[MAX_SLOTS], empty[MAX_SLOTS], raw_full[4], raw_empty[4], s_ready[2], p_ready[2][2], o_done, q_ready, drained;
    float crow[R];
    uint64_t turns[64]; // a lane's own entry is no broadcast: not from the constant bank
    uint32_t tmem;
    int abort;
};

// one CTA's pieces in order; every role walks them by itself
struct Walk {
    KqSeq sq;
    int s, kh, tile, tiles, ub, take, n_units;
    int2 keys;
    long long u, u1, uo;
    __device__ void start(const KqAttnArgs &a, const KqRun &run) {
        u = run.u0;
        u1 = run.u1;
        s = run.s;
        if (u >= u1) return;
        sq = kq_seq(a, s);
        kh = (int)kq_div(run.off, run.per_head);
        uo = run.off - kh * run.per_head;
        tiles = kq_tiles<R>(a, sq.t);
        // the tile that the run begins in: a lane counts one of 32
        const int lane = threadIdx.x & 31;
        for (tile = 0; tile < tiles; tile += 32) {
            const int mine = tile + lane < tiles ? kq_units<BK>(kq_tile_keys<R>(a, sq, tile + lane)) + kq_setup<R> : 0;
            int upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            const unsigned past = __ballot_sync(0xffffffffu, (long long)upto > uo);
            if (past) {
                const int l = __ffs(past) - 1;
                uo -= __shfl_sync(0xffffffffu, upto - mine, l);
                tile += l;
                break;
            }
            uo -= __shfl_sync(0xffffffffu, upto, 31);
        }
    }
    // the next piece; false: no more
    __device__ bool next(const KqAttnArgs &a) {
        for (;; done()) {
            if (u >= u1) return false;
            while (tile >= tiles) {
                tile = 0;
                if (++kh >= a.c.n_kv) {
                    kh = 0;
                    do {
                        if (++s >= a.b.n_seq) return false;
                        sq = kq_seq(a, s);
                    } while (sq.t == 0);
                    tiles = kq_tiles<R>(a, sq.t);
                }
            }
            keys = kq_tile_keys<R>(a, sq, tile);
            n_units = kq_units<BK>(keys);
            const int part = (int)min((long long)n_units + kq_setup<R> - uo, u1 - u);
            ub = max(0, (int)uo - kq_setup<R>);
            take = max(0, (int)uo + part - kq_setup<R>) - ub;
            u += part;
            if (take > 0) return true; // else the item is the next CTA's
        }
    }
    __device__ void done() {
        tile++;
        uo = 0;
    }
};

template <bool F8> __device__ __forceinline__ void less_registers() {
    if (F8) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
}
// codes of 8 dimensions as f16 numbers times the block's scale
__device__ __forceinline__ uint4 decode8(uint32_t lo, uint32_t hi, __half2 s) {
    uint4 v;
    kq_e4m3x4_h2(lo, v.x, v.y);
    kq_e4m3x4_h2(hi, v.z, v.w);
    auto scaled = [&](uint32_t &h) {
        const __half2 r = __hmul2(*reinterpret_cast<const __half2 *>(&h), s);
        h = *reinterpret_cast<const uint32_t *>(&r);
    };
    scaled(v.x), scaled(v.y), scaled(v.z), scaled(v.w);
    return v;
}

// T: the activations' type; f32 and f16 queries in two f16 parts, probabilities of f32 results in two
template <int HD, bool F8, typename T>
__global__ void __launch_bounds__(F8 ? 512 : 384, 1)
    pages_prompt_kernel(const __grid_constant__ KqAttnArgs a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, int box_rows) {
    constexpr int QS = std::is_same<T, __nv_bfloat16>::value ? 1 : 2, PS = std::is_same<T, float>::value ? 2 : 1;
    constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
    using L = Layout<HD, F8, QS>;
    constexpr int NS = L::NS, NR = L::NR > 0 ? L::NR : 1, NT = F8 ? 512 : 384;
    extern __shared__ __align__(1024) uint8_t sm_raw[];
    uint8_t *sm = sm_raw + ((1024u - (smem_u32(sm_raw) & 1023u)) & 1023u);
    __shared__ Shared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid < HD / 2) sh.turns[tid] = a.turns.f[tid];
    if (tid == 0) {
        auto init = [](uint64_t &b, int n) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&b)), "r"(n)); };
        for (int i = 0; i < MAX_SLOTS; i++) {
            init(sh.full[i], F8 ? 128 : 1);
            init(sh.empty[i], 1);
        }
        for (int i = 0; i < 4; i++) {
            init(sh.raw_full[i], 1);
            init(sh.raw_empty[i], 128);
        }
        for (int i = 0; i < 2; i++) {
            init(sh.s_ready[i], 1);
            init(sh.p_ready[i][0], 128); // probabilities of the first 64 keys
            init(sh.p_ready[i][1], 128); // and of the others
        }
        init(sh.o_done, 1);
        init(sh.drained, 1);
        init(sh.q_ready, NSOFT);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        sh.abort = 0;
    }
    KQ_PDL_ENTER();
    // behind the dependency wait: a CTA that starts early must not hold columns that its predecessor still has to allocate
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    before_sync();
    __syncthreads();
    after_sync();
    const uint32_t tmem = sh.tmem;
    volatile int *abort = &sh.abort;
    auto wait = [&](uint64_t &bar, uint32_t parity, int code) { return tc_wait(smem_u32(&bar), parity, abort, &g_pages_error, code, LIMIT); };
    const KqRun run = kq_find_run<R, BK, NT>(a);
    Walk w;
    w.start(a, run);
    const int bpp = a.c.page / KQ_PAGE_BLOCK;
    int4 meta = make_int4(0, 0, 0, 0), meta2 = meta;

    // registers: the launch's 384 x 168 as 256 x 208 + 128 x 88, or 512 x 128 as 256 x 184 + 256 x 72
    if (warp == 8) {
        less_registers<F8>();
        // ---------------------------------------------------------------- products: all lanes run the loop, one issues
        const bool lead = tc_elect();
        auto wait_all = [&](uint64_t &bar, uint32_t parity, int code) { return __all_sync(0xffffffffu, wait(bar, parity, code)) != 0; };
        const uint32_t ring = smem_u32(sm + L::RING);
        const uint64_t dq = tc_desc(smem_u32(sm), 16, 1024), dk = tc_desc(ring, 16, 1024), dv = tc_desc(ring, HALF, 1024);
        uint32_t pieces = 0, units = 0, ks = 0, kph = 0; // slot of the next tile of the ring and the parity of its round
        bool ok = true;
        bool both = true; // the second tile has rows
        auto scores = [&](int half, uint32_t slot) {
            if (!lead || !ok || (half && !both)) return;
            const uint64_t b = dk + slot * (L::TILE / 16);
#pragma unroll
            for (int p = 0; p < QS; p++)
#pragma unroll
                for (int s = 0; s < HD / 16; s++)
                    tc_mma_ss(tmem + COL_S + 128 * half, dq + (2 * p + half) * (L::TILE / 16) + step_k(s), b + step_k(s), tc_idesc(128, BK, false, false), p + s > 0);
        };
        auto values = [&](int half, uint32_t slot, bool first) { // the first 64 keys' product begins while the other probabilities are worked out
            const uint64_t b = dv + slot * (L::TILE / 16);
#pragma unroll
            for (int x = 0; x < 2; x++) {
                ok = wait_all(sh.p_ready[half][x], units & 1, 3) && ok;
                after_sync();
                if (lead && ok && (!half || both)) {
#pragma unroll
                    for (int p = 0; p < PS; p++)
#pragma unroll
                        for (int s = 4 * x; s < 4 * x + 4; s++)
                            tc_mma_ts(tmem + COL_O + 128 * half, tmem + COL_S + 128 * half + 64 * x + 32 * p + 8 * (s & 3), b + step_mn(s), tc_idesc(128, HD, false, true),
                                      x + p + s > 0 ? 1u : first ? 0u : 1u);
                }
                __syncwarp();
            }
        };
        auto next = [&](uint32_t &slot, uint32_t &ph) {
            if (++slot == NS) slot = 0, ph ^= 1;
        };
        while (w.next(a)) {
            both = w.sq.t * a.G - w.tile * R > 128;
            ok = wait_all(sh.q_ready, pieces & 1, 1) && ok;
            ok = wait_all(sh.full[ks], kph, 2) && ok;
            after_sync();
            scores(0, ks);
            if (lead) tc_commit(smem_u32(&sh.s_ready[0]));
            scores(1, ks);
            if (lead) {
                tc_commit(smem_u32(&sh.s_ready[1]));
                tc_commit(smem_u32(&sh.empty[ks]));
            }
            __syncwarp();
            for (int i = 0; i < w.take; i++) {
                const bool more = i + 1 < w.take, first = i == 0;
                uint32_t vs = ks, vph = kph;
                next(vs, vph);
                ks = vs, kph = vph;
                next(ks, kph);
                ok = wait_all(sh.full[vs], vph, 4) && ok;
                values(0, vs, first);
                if (more) {
                    ok = wait_all(sh.full[ks], kph, 5) && ok;
                    after_sync();
                    scores(0, ks);
                    if (lead) tc_commit(smem_u32(&sh.s_ready[0]));
                    __syncwarp();
                }
                values(1, vs, first);
                if (lead) tc_commit(smem_u32(&sh.empty[vs]));
                if (more) {
                    scores(1, ks);
                    if (lead) {
                        tc_commit(smem_u32(&sh.s_ready[1]));
                        tc_commit(smem_u32(&sh.empty[ks]));
                    }
                }
                __syncwarp();
                units++;
            }
            if (lead) tc_commit(smem_u32(&sh.o_done));
            __syncwarp();
            pieces++;
            w.done();
        }
        if (!ok && lead) { // products in flight end before TMEM is freed
            tc_commit(smem_u32(&sh.drained));
            kq_mbar_wait(smem_u32(&sh.drained), 0, KQ_WAIT_LIMIT_NS);
        }
        __syncwarp();
    } else if (warp == 9) {
        less_registers<F8>();
        // ---------------------------------------------------------------- copies: a lane per box
        const int boxes = BK / box_rows, halves = F8 ? 1 : HD / 64, box = lane / halves, half = lane % halves;
        uint32_t tile_n = 0;
        while (w.next(a)) {
            const int seen = a.window > 0 ? max(0, w.sq.pos(w.tile * R / a.G) - a.window + 1) : 0; // before this no row sees anything
            auto look_up = [&](int i) { // page of this lane's box of unit i, -1: nothing to fetch
                const int key = w.keys.x + (w.ub + i) * BK + box * box_rows;
                return i < w.take && box < boxes && key < w.keys.y && key + box_rows > seen ? kq_page_of(a.c, w.s, key) : -1;
            };
            int id = look_up(0);
            for (int i = 0; i < w.take; i++) {
                const int key = w.keys.x + (w.ub + i) * BK + box * box_rows, place = key % a.c.page, next = look_up(i + 1);
                for (int kv = 0; kv < 2; kv++, tile_n++) {
                    if constexpr (F8) {
                        uint64_t &full = sh.raw_full[tile_n % NR];
                        wait(sh.raw_empty[tile_n % NR], ((tile_n / NR) & 1) ^ 1, 7);
                        const uint32_t n = __popc(__ballot_sync(0xffffffffu, id >= 0)), bytes = box_rows * HD;
                        if (lane == 0) expect(smem_u32(&full), *abort ? 0 : n * bytes);
                        __syncwarp();
                        if (id >= 0 && !*abort)
                            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                                             smem_u32(sm + L::RAWS + (tile_n % NR) * L::RAW + box * bytes)),
                                         "l"((kv ? a.c.v : a.c.k) + (int64_t)id * a.c.page_bytes + ((int64_t)w.kh * a.c.page + place) * HD), "r"(bytes), "r"(smem_u32(&full))
                                         : "memory");
                    } else {
                        uint64_t &full = sh.full[tile_n % NS];
                        wait(sh.empty[tile_n % NS], ((tile_n / NS) & 1) ^ 1, 7);
                        if (lane == 0) expect(smem_u32(&full), *abort ? 0 : L::TILE);
                        __syncwarp();
                        if (box < boxes && !*abort) // a page that is not there comes as zeros: its coordinate is past the end
                            asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                                             smem_u32(sm + L::RING + (tile_n % NS) * L::TILE + half * HALF + box * box_rows * 128)),
                                         "l"(kv ? &vmap : &kmap), "r"(64 * half), "r"(w.kh * a.c.page + place), "r"(id >= 0 ? id : (int)a.c.n_pages), "r"(smem_u32(&full))
                                         : "memory");
                    }
                    __syncwarp();
                }
                id = next;
            }
            w.done();
        }
        if (*abort && lane == 0) // what is in flight must land before the CTA goes away
            for (int i = 0; i < (F8 ? NR : NS); i++) {
                uint64_t &b = F8 ? sh.raw_full[i] : sh.full[i];
                kq_mbar_wait(smem_u32(&b), 0u, KQ_WAIT_LIMIT_NS);
                kq_mbar_wait(smem_u32(&b), 1u, KQ_WAIT_LIMIT_NS);
            }
        __syncwarp();
    } else if (F8 && warp >= 12) {
        less_registers<F8>();
        // ---------------------------------------------------------------- e4m3 rows to the f16 tile: a thread per position
        const int c = tid - 384;
        uint32_t tile_n = 0;
        while (w.next(a)) {
            const int seen = a.window > 0 ? max(0, w.sq.pos(w.tile * R / a.G) - a.window + 1) : 0;
            auto look_up = [&](int i) {
                const int key = w.keys.x + (w.ub + i) * BK + c;
                return i < w.take && key < w.keys.y && key >= seen ? kq_page_of(a.c, w.s, key) : -1;
            };
            auto scales = [&](int i, int id) { // of the position's block
                if (id < 0) return make_float2(0.f, 0.f);
                const int64_t at = ((int64_t)id * a.c.n_kv + w.kh) * bpp + (w.keys.x + (w.ub + i) * BK + c) % a.c.page / KQ_PAGE_BLOCK;
                return make_float2(a.c.ks[at], a.c.vs[at]);
            };
            int id = look_up(0), id1 = look_up(1); // pages two units ahead, scales one: their loads are under way while a unit is converted
            float2 sc = scales(0, id);
            for (int i = 0; i < w.take; i++) {
                const int id2 = look_up(i + 2);
                const float2 sc1 = scales(i + 1, id1);
#pragma unroll 1
                for (int kv = 0; kv < 2; kv++, tile_n++) {
                    constexpr int NC = HD / 16; // 16-byte chunks of a raw row; taken in an order that keeps eight rows off each other's banks
                    uint4 raw[NC];
                    wait(sh.raw_full[tile_n % NR], (tile_n / NR) & 1, 8);
                    const uint8_t *src = sm + L::RAWS + (tile_n % NR) * L::RAW + c * HD;
#pragma unroll
                    for (int j = 0; j < NC; j++) raw[j] = id >= 0 ? *reinterpret_cast<const uint4 *>(src + ((j + c) % NC) * 16) : make_uint4(0, 0, 0, 0);
                    arrive(smem_u32(&sh.raw_empty[tile_n % NR]));
                    const __half2 s = __float2half2_rn(kv ? sc.y : sc.x);
                    wait(sh.empty[tile_n % NS], ((tile_n / NS) & 1) ^ 1, 9);
                    uint8_t *dst = sm + L::RING + (tile_n % NS) * L::TILE + c * 128;
#pragma unroll
                    for (int j = 0; j < NC; j++) {
                        const int o = 2 * ((j + c) % NC); // the first of two chunks of 8 dimensions
                        uint8_t *d = dst + (o >> 3) * HALF;
                        *reinterpret_cast<uint4 *>(d + (((o & 7) ^ (c & 7)) << 4)) = decode8(raw[j].x, raw[j].y, s);
                        *reinterpret_cast<uint4 *>(d + ((((o & 7) + 1) ^ (c & 7)) << 4)) = decode8(raw[j].z, raw[j].w, s);
                    }
                    fence_async();
                    arrive(smem_u32(&sh.full[tile_n % NS]));
                }
                id = id1;
                id1 = id2;
                sc = sc1;
            }
            w.done();
        }
    } else if (warp < 8) {
        if (F8) asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
        else asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        // ---------------------------------------------------------------- queries, softmax, results: a thread per row
        const int half = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t tl = tmem + ((uint32_t)((warp & 3) * 32) << 16), ts = tl + COL_S + 128 * half, to = tl + COL_O + 128 * half;
        uint32_t pieces = 0, units = 0;
        // f16 values that no row sees may hold anything: they must not meet a probability of 0.  The first half's threads have a position of the tile each
        auto hide_values = [&](int key0, int seen) {
            if (F8 || half || (key0 + BK <= w.keys.y && key0 >= seen)) return;
            const uint32_t v = 2 * units + 1;
            wait(sh.full[v % NS], (v / NS) & 1, 11);
            if (key0 + row >= w.keys.y || key0 + row < seen) {
                uint8_t *d = sm + L::RING + (v % NS) * L::TILE + row * 128;
#pragma unroll
                for (int j = 0; j < HD / 8; j++) *reinterpret_cast<uint4 *>(d + (j >> 3) * HALF + (j & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            __syncwarp();
            fence_async();
        };
        while (w.next(a)) {
            const int row0 = w.tile * R + 128 * half; // of this half, within the sequence and KV head
            const int seen = a.window > 0 ? max(0, w.sq.pos(w.tile * R / a.G) - a.window + 1) : 0; // before this no row sees anything
            if (row0 + (warp & 3) * 32 >= w.sq.t * a.G) { // none of the warp's rows is one: what the products make of its places is not looked at
                arrive(smem_u32(&sh.q_ready));
                for (int i = 0; i < w.take; i++, units++) {
                    wait(sh.s_ready[half], units & 1, 10);
                    hide_values(w.keys.x + (w.ub + i) * BK, seen);
                    arrive(smem_u32(&sh.p_ready[half][0]));
                    arrive(smem_u32(&sh.p_ready[half][1]));
                }
                wait(sh.o_done, pieces & 1, 12);
                pieces++;
                w.done();
                continue;
            }
            // ---- queries: a warp's 32 rows are copied to where they will stand as f16 parts (which is as large), all in flight together, and then turned
            // in place, eight at a time.  The angles of the warp's tokens (rows of one share them) are worked out meanwhile, in a loop of their own: in line with the rows they
            // are 60 KB of code, and fetching it took four times as long as running it; out of line the calls spill what the rows hold.
            constexpr int P = HD / 64, NB = 8, CH = HD * (int)sizeof(T) / 16; // 16-byte chunks of a row
            static_assert(NB == 8, "rows are swizzled by eights");
            const bool split = a.turns.on && a.turns.neox;
            const int wrow = (warp & 3) * 32, tok0 = (row0 + wrow) / a.G, h0 = row0 + wrow - tok0 * a.G;
            auto raw_at = [&](int r, int c) { // chunk c of row r of this half
                const int b = c >> 3, part = HD == 128 ? b >> 1 : b;
                return sm + (2 * part + half) * L::TILE + (HD == 128 ? (b & 1) * HALF : 0) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
            };
            {
                constexpr int STEP = 32 / CH; // rows of one copy of the warp
                const int c = lane % CH, left = (w.sq.t - tok0) * a.G - h0; // rows of the sequence and KV head from the warp's first on
                int ch = h0 + lane / CH;
                const T *src = (const T *)a.q + (int64_t)(w.sq.row0 + tok0) * a.q_stride + (int64_t)(w.kh * a.G + ch) * HD + c * (16 / (int)sizeof(T));
                const int64_t turn = a.q_stride - (int64_t)a.G * HD; // from behind a token's heads to the next token's
#pragma unroll 4
                for (int r = lane / CH; r < 32; r += STEP, ch += STEP, src += STEP * HD) {
                    while (ch >= a.G) ch -= a.G, src += turn;
                    const bool there = r < left;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(raw_at(wrow + r, c))), "l"(there ? src : (const T *)a.q), "r"(there ? 16 : 0) : "memory");
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            float4 cs[33]; // of the lane's pairs, by token; in local memory
            const int toks = min((h0 + 31) / a.G + 1, w.sq.t - tok0);
#pragma unroll 2
            for (int i = 0; i < toks; i++) {
                float2 x = make_float2(1.f, 0.f), y = x;
                if (a.turns.on) {
                    x = kq_turn(sh.turns[P * lane], w.sq.pos(tok0 + i));
                    y = P == 2 ? kq_turn(sh.turns[P * lane + P - 1], w.sq.pos(tok0 + i)) : x;
                }
                cs[i] = make_float4(x.x, x.y, y.x, y.y);
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncwarp();
            int tok = 0, h = h0; // token of the next row, counted from tok0, and its head
            // the lane's pairs are P lane + u: dimensions (pair, pair + HD / 2) or (2 pair, 2 pair + 1)
#pragma unroll 1
            for (int rb = 0; rb < min(32, (w.sq.t - tok0) * a.G - h0); rb += NB) { // places behind the last row keep what they hold: nothing looks at them
                float x[NB][P][2];
                float2 c[NB][P];
                uint8_t *rows8 = sm + half * L::TILE + (wrow + rb) * 128; // eight rows, the place of each among eight is its swizzle
                auto at8 = [&](int k, int d) { // element d of row k
                    constexpr int PER = 16 / (int)sizeof(T);
                    const int c = d / PER, b = c >> 3;
                    return reinterpret_cast<const T *>(rows8 + (HD == 128 ? (b >> 1) * (2 * L::TILE) + (b & 1) * HALF : b * (2 * L::TILE)) + k * 128 + (((c & 7) ^ k) << 4)) + d % PER;
                };
                auto pair_at = [&](int k, int d) { return kq_ld2(at8(k, d)); };
                auto one_at = [&](int k, int d) { return kq_ld1(at8(k, d)); };
#pragma unroll
                for (int k = 0; k < NB; k++) {
                    const float4 v = tok < toks ? cs[tok] : make_float4(1.f, 0.f, 1.f, 0.f);
                    c[k][0] = make_float2(v.x, v.y);
                    c[k][P - 1] = P == 2 ? make_float2(v.z, v.w) : c[k][0];
                    if (++h == a.G) h = 0, tok++;
                }
#pragma unroll
                for (int k = 0; k < NB; k++) {
                    if (split && P == 2) {
                        const float2 v0 = pair_at(k, 2 * lane), v1 = pair_at(k, HD / 2 + 2 * lane);
                        x[k][0][0] = v0.x, x[k][P - 1][0] = v0.y, x[k][0][1] = v1.x, x[k][P - 1][1] = v1.y;
                    } else if (split) {
                        x[k][0][0] = one_at(k, lane);
                        x[k][0][1] = one_at(k, HD / 2 + lane);
                    } else {
#pragma unroll
                        for (int u = 0; u < P; u++) {
                            const float2 v = pair_at(k, 2 * (P * lane + u));
                            x[k][u][0] = v.x, x[k][u][1] = v.y;
                        }
                    }
                }
                __syncwarp(); // every lane has its elements of the rows
                float amax[NB];
#pragma unroll
                for (int k = 0; k < NB; k++) {
                    amax[k] = 0.f;
#pragma unroll
                    for (int u = 0; u < P; u++) {
                        const float v0 = x[k][u][0], v1 = x[k][u][1];
                        x[k][u][0] = v0 * c[k][u].x - v1 * c[k][u].y;
                        x[k][u][1] = v0 * c[k][u].y + v1 * c[k][u].x;
                        amax[k] = fmaxf(amax[k], fmaxf(fabsf(x[k][u][0]), fabsf(x[k][u][1])));
                    }
                }
#pragma unroll
                for (int k = 0; k < NB; k++) amax[k] = kq_warp_top(amax[k]);
#pragma unroll
                for (int k = 0; k < NB; k++) {
                    const int r = (warp & 3) * 32 + rb + k;
                    const uint32_t e = min(max(__float_as_uint(amax[k]) >> 23, 1u), 252u);
                    const float f = amax[k] > 0.f ? __uint_as_float((254u - e) << 23) : 1.f;
                    if (lane == 0) sh.crow[128 * half + r] = fmaxf(amax[k] > 0.f ? a.scale_log2 * __uint_as_float(e << 23) : a.scale_log2, 1.2e-38f); // not 0: a hidden score times it is -inf
                    auto put = [&](int d, float v0, float v1, bool two) { // dimension d (and d + 1)
#pragma unroll
                        for (int p = 0; p < QS; p++) {
                            uint8_t *at = rows8 + p * (2 * L::TILE) + (d >> 6) * HALF + k * 128 + ((((d >> 3) & 7) ^ k) << 4) + (d & 7) * 2;
                            const uint32_t hi = kq_h2(v0, v1), v = p ? kq_h2_low(v0, v1, hi) : hi;
                            if (two) *reinterpret_cast<uint32_t *>(at) = v;
                            else *reinterpret_cast<uint16_t *>(at) = (uint16_t)v;
                        }
                    };
                    if (split && P == 2) {
                        put(2 * lane, x[k][0][0] * f, x[k][P - 1][0] * f, true);
                        put(HD / 2 + 2 * lane, x[k][0][1] * f, x[k][P - 1][1] * f, true);
                    } else if (split) {
                        put(lane, x[k][0][0] * f, 0.f, false);
                        put(HD / 2 + lane, x[k][0][1] * f, 0.f, false);
                    } else {
#pragma unroll
                        for (int u = 0; u < P; u++) put(2 * (P * lane + u), x[k][u][0] * f, x[k][u][1] * f, true);
                    }
                }
            }
            fence_async();
            arrive(smem_u32(&sh.q_ready));
            __syncwarp();
            const float crow = sh.crow[128 * half + row];
            const bool my_row_ok = (row0 + row) / a.G < w.sq.t;
            const int my_tok = min((row0 + row) / a.G, w.sq.t - 1), lim = w.sq.p0 < 0 ? -1 : w.sq.pos(my_tok); // last position this row sees
            const int lim_lo = w.sq.pos(min(row0 / a.G, w.sq.t - 1)), lim_hi = w.sq.pos(min((row0 + 127) / a.G, w.sq.t - 1)); // of the half's rows
            auto look_up = [&](int i) { // is the lane's block (of 32 from unit i on) there
                const int key = w.keys.x + (w.ub + i) * BK + KQ_PAGE_BLOCK * lane;
                return key < w.keys.y ? kq_page_of(a.c, w.s, key) : -1;
            };
            uint32_t there = 0;
            int ahead = look_up(0);
            const int slot = 2 * blockIdx.x + (w.ub == 0 ? 1 : 0); // of a piece that is not the whole item
            // sums put aside: four columns of all rows next to one another, so that a warp's lanes write one run
            float *aside = a.part + (int64_t)gridDim.x * 2 * R * (HD + 2) + (int64_t)blockIdx.x * R * HD + 4 * (128 * half + row);
            int joined = 0;     // units in O since it was put aside
            float last_l = 0.f; // what the last one added to l
            float m = -INFINITY, l = 0.f;
            float2 put = make_float2(-INFINITY, 0.f); // of what was put aside: the maximum that it goes by, and its l
            // bf16, which seldom puts anything aside, keeps it in memory (2048 rows at 6144: 321 us, in registers 331, never 317; f16 421 and 410)
            auto put_at = [&] { return reinterpret_cast<float2 *>(a.part + (int64_t)gridDim.x * R * (2 * (HD + 2) + HD)) + (int64_t)blockIdx.x * R + 128 * half + row; };
            // the row's O so far: what the tensor cores have summed and what was put aside before; as 32 columns a time
            auto total = [&](int k, uint32_t *o, float2 put) {
                tmem_ld32(to + 32 * k, o);
                tmem_ld_wait();
                if (put.x != -INFINITY) {
                    const float f = kq_ex2(put.x - m);
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const float4 v = *reinterpret_cast<const float4 *>(aside + (8 * k + j / 4) * (4 * R));
                        o[j] = __float_as_uint(fmaf(v.x, f, __uint_as_float(o[j])));
                        o[j + 1] = __float_as_uint(fmaf(v.y, f, __uint_as_float(o[j + 1])));
                        o[j + 2] = __float_as_uint(fmaf(v.z, f, __uint_as_float(o[j + 2])));
                        o[j + 3] = __float_as_uint(fmaf(v.w, f, __uint_as_float(o[j + 3])));
                    }
                }
                __syncwarp();
            };
            for (int i = 0; i < w.take; i++, units++) {
                if ((i & 3) == 0) {
                    there = __ballot_sync(0xffffffffu, ahead >= 0);
                    ahead = look_up(i + 4);
                }
                const uint32_t blocks = (there >> (8 * (i & 3))) & 0xff;
                const int key0 = w.keys.x + (w.ub + i) * BK;
                wait(sh.s_ready[half], units & 1, 10);
                __syncwarp(); // what reads and writes TMEM takes whole warps
                after_sync(); // S was issued behind the products before: O is at rest
                if (BF ? i > 0 && i % FLUSH<T> == 0 : joined == FLUSH<T> || (PS == 2 && __any_sync(0xffffffffu, last_l > 0.f && l > DOMINATED * last_l))) {
                    if (BF && i > FLUSH<T>) put = *put_at();
#pragma unroll
                    for (int k = 0; k < HD / 32; k++) {
                        uint32_t o[32];
                        total(k, o, put);
#pragma unroll
                        for (int j = 0; j < 32; j += 4)
                            *reinterpret_cast<uint4 *>(aside + (8 * k + j / 4) * (4 * R)) = make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]);
#pragma unroll
                        for (int j = 0; j < 32; j++) o[j] = 0;
                        if (!*abort) tmem_st32(to + 32 * k, o);
                    }
                    tmem_st_wait();
                    put.y = l + (put.x != -INFINITY ? put.y * kq_ex2(put.x - m) : 0.f);
                    put.x = m;
                    l = 0.f;
                    joined = 0;
                    if (BF) {
                        *put_at() = put;
                        put = make_float2(-INFINITY, 0.f);
                    }
                }
                joined++;
                const bool masked = blocks != 0xff || key0 + BK - 1 > lim_lo || (a.window > 0 && key0 <= lim_hi - a.window);
                const int last = lim - key0, first = a.window > 0 ? last - a.window + 1 : -0x40000000;
                auto mask = [&](uint32_t *s, int c) {
                    // bit j: score j of the chunk is seen
                    const int hi = last - 32 * c, lo = first - 32 * c;
                    uint32_t see = hi >= 31 ? 0xffffffffu : hi < 0 ? 0u : (2u << hi) - 1u;
                    if (lo > 0) see &= lo > 31 ? 0u : 0xffffffffu << lo;
                    if (!(blocks >> (2 * c) & 1)) see &= 0xffff0000u;
                    if (!(blocks >> (2 * c + 1) & 1)) see &= 0x0000ffffu;
#pragma unroll
                    for (int j = 0; j < 32; j++)
                        if (!(see >> j & 1)) s[j] = 0xff800000u; // -inf
                };
                uint32_t s[4][32];
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}; // a NaN stays: the whole row is NaN from there on
#pragma unroll
                for (int c = 0; c < 4; c++) tmem_ld32(ts + 32 * c, s[c]);
                tmem_ld_wait();
                if (masked) {
#pragma unroll
                    for (int c = 0; c < 4; c++) mask(s[c], c);
                }
#pragma unroll
                for (int c = 0; c < 4; c++)
#pragma unroll
                    for (int j = 0; j < 32; j += 2) mx[(j >> 1) & 3] = max3(mx[(j >> 1) & 3], __uint_as_float(s[c][j]), __uint_as_float(s[c][j + 1]));
                const float top = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]) * crow;
                const bool grown = !(top <= m + GROWTH) || m == -INFINITY; // the first tile, or a maximum that would make probabilities too large
                if (__any_sync(0xffffffffu, grown)) {
                    const float mn = grown ? max3(m, top, top) : m, alpha = mn == m ? 1.f : kq_ex2(m - mn);
                    m = mn;
                    if (i > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
                        l *= alpha;
#pragma unroll
                        for (int k = 0; k < HD / 32; k++) {
                            uint32_t o[32];
                            tmem_ld32(to + 32 * k, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int j = 0; j < 32; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
                            if (!*abort) tmem_st32(to + 32 * k, o);
                        }
                    }
                }
                const float sub = m == -INFINITY ? 0.f : m - PEAK;
                hide_values(key0, seen);
                uint64_t sums[2] = {0, 0}; // f32: of the steps of a chunk; bf16: of all keys, in two runs
                float rounded[4] = {0.f, 0.f, 0.f, 0.f}; // f16's
                const float l_before = l;
                uint32_t lo_even[PS == 2 ? 16 : 1];
                const uint64_t crow2 = pack2(crow, crow), nsub2 = pack2(-sub, -sub);
                // a chunk's probabilities go over scores that have been read: those of keys 0 .. 63 to columns 0 .. 31 (second parts 32 .. 63) ...
#pragma unroll
                for (int h64 = 0; h64 < 2; h64++) {
                    uint32_t hi[16], lo[PS == 2 ? 16 : 1];
                    float cuts = 0.f; // of the second parts' steps
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int c = 2 * h64 + e;
                        uint32_t(&x)[32] = s[c];
#pragma unroll
                        for (int j = 0; j < 16; j++) {
                            uint64_t v = fma2(pack2(__uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1])), crow2, nsub2);
                            // results of 8 bits: 3 of 8 exponentials on the FMA pipe, so that neither it nor the special-function unit decides alone
                            // (4096 rows behind 12288 positions: 1509, 1480, 1460, 1437 us for 0, 1, 2, 3 of 8, when these were tried)
                            v = BF && j % 8 < POLY ? exp2_poly(v) : exp2_sfu(v);
                            if (BF) sums[j & 1] = add2(sums[j & 1], v);
                            const float2 p = unpack2(v);
                            hi[j] = kq_h2(p.x, p.y);
                            // f16: the divisor is the sum of the weights as O has them, rounded, so that one weight's rounding is not the result's.  (Two parts
                            // as in f32 take 2048 rows at 6144 from 385 to 484 us, for results 1.01 instead of 1.13 half steps off.)
                            if (PS == 1 && !BF) {
                                rounded[j & 1] = add_f16(rounded[j & 1], hi[j]);
                                rounded[2 + (j & 1)] = add_f16(rounded[2 + (j & 1)], hi[j] >> 16);
                            }
                            if (PS == 2) {
                                sums[j >> 3] = add2(sums[j >> 3], v);
                                const uint32_t rest = kq_h2_low(p.x, p.y, hi[j]);
                                if (e == 0) lo_even[PS == 2 ? j : 0] = rest;
                                else lo[PS == 2 ? j : 0] = rest;
                            }
                        }
                        if (PS == 2) {
#pragma unroll
                            for (int g = 0; g < 2; g++) {
                                const float2 v = unpack2(sums[g]);
                                const float sum = v.x + v.y;
                                l = __fadd_rz(l, sum);
                                // second parts are 2^-12 of the first at most, and there are none where a step's sum is one of f16 numbers (which leave low bits 0)
                                if (sum >= l * 0x1p-13f && (__float_as_uint(sum) & 0x7ff)) cuts += CUT_HALF_BIT;
                                sums[g] = 0;
                            }
                            if (e) l = fmaf(l, -cuts, l);
                        }
                        if (!*abort) {
                            tmem_st16(ts + 64 * h64 + 16 * e, hi);
                            if (PS == 2 && e) { // columns 32 .. 63 of the half are free once its second chunk has been read
                                tmem_st16(ts + 64 * h64 + 32, lo_even);
                                tmem_st16(ts + 64 * h64 + 48, lo);
                            }
                        }
                    }
                    tmem_st_wait();
                    before_sync();
                    arrive(smem_u32(&sh.p_ready[half][h64]));
                }
                if (PS == 2) last_l = l - l_before;
                else {
                    const float2 v = unpack2(add2(sums[0], sums[1]));
                    l += BF ? v.x + v.y : (rounded[0] + rounded[1]) + (rounded[2] + rounded[3]);
                }
            }
            // ---- results
            wait(sh.o_done, pieces & 1, 12);
            __syncwarp();
            after_sync();
            if (BF && w.take > FLUSH<T>) put = *put_at();
            if (put.x != -INFINITY) l = fmaf(put.y, kq_ex2(put.x - m), l);
            const bool whole = w.ub == 0 && w.take == w.n_units, ok = my_row_ok && !*abort;
            const float inv = m == -INFINITY ? 0.f : whole ? 1.f / l : 1.f; // a row that saw nothing is 0
            // 32 columns a time through the warp's part of the queries' room, so that a store writes whole lines of 4 rows
            uint8_t *turn = sm + half * L::TILE + (warp & 3) * 4096;
            const int cr = lane >> 3, cc = lane & 7; // row of four and 16-byte chunk of a store
            int64_t to_row[8]; // where this lane's rows go, -1: nowhere
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int r = 4 * j + cr, rr = row0 + (warp & 3) * 32 + r, tok = rr / a.G, h = rr - tok * a.G; // r: of the warp's 32 rows
                to_row[j] = tok >= w.sq.t || *abort ? -1 : whole ? (int64_t)(w.sq.row0 + tok) * a.out_stride + (int64_t)(w.kh * a.G + h) * HD + 4 * cc
                                                        : (int64_t)slot * R * (HD + 2) + (int64_t)(128 * half + (warp & 3) * 32 + r) * HD + 4 * cc;
            }
#pragma unroll 1
            for (int k = 0; k < HD / 32; k++) {
                uint32_t o[32];
                __syncwarp();
                total(k, o, put);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    float4 v;
                    v.x = __uint_as_float(o[4 * j]) * inv, v.y = __uint_as_float(o[4 * j + 1]) * inv, v.z = __uint_as_float(o[4 * j + 2]) * inv, v.w = __uint_as_float(o[4 * j + 3]) * inv;
                    if (m == -INFINITY) v = make_float4(0.f, 0.f, 0.f, 0.f);
                    *reinterpret_cast<float4 *>(turn + lane * 128 + ((j ^ (lane & 7)) << 4)) = v;
                }
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int r = 4 * j + cr;
                    const float4 v = *reinterpret_cast<const float4 *>(turn + r * 128 + ((cc ^ (r & 7)) << 4));
                    if (to_row[j] < 0) continue;
                    if (!whole) *reinterpret_cast<float4 *>(a.part + to_row[j] + 32 * k) = v;
                    else {
                        T *out = (T *)a.out + to_row[j] + 32 * k;
                        if constexpr (sizeof(T) == 4) *reinterpret_cast<float4 *>(out) = v;
                        else if constexpr (std::is_same<T, __half>::value) *reinterpret_cast<uint2 *>(out) = make_uint2(kq_h2(v.x, v.y), kq_h2(v.z, v.w));
                        else {
                            const __nv_bfloat162 b[2] = {__floats2bfloat162_rn(v.x, v.y), __floats2bfloat162_rn(v.z, v.w)};
                            *reinterpret_cast<uint2 *>(out) = *reinterpret_cast<const uint2 *>(b);
                        }
                    }
                }
            }
            __syncwarp(); // the next item's queries go where the rows went through
            if (!whole && ok) {
                float *ml = a.part + (int64_t)slot * R * (HD + 2) + (int64_t)R * HD + 2 * (128 * half + row);
                *reinterpret_cast<float2 *>(ml) = make_float2(m, l);
            }
            if (w.ub == 0 && !whole) {
                meta = make_int4(1 + (int)kq_div(w.n_units - w.take + (run.u1 - run.u0) - 1, run.u1 - run.u0), w.kh, w.tile, 0);
                meta2 = make_int4(w.sq.row0, w.sq.t, 0, 0);
            }
            before_sync();
            pieces++;
            w.done();
        }
        if (tid == 0) {
            a.meta[2 * blockIdx.x] = meta;
            a.meta[2 * blockIdx.x + 1] = meta2;
        }
    } else less_registers<F8>();
    before_sync();
    __syncthreads();
    if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// joins the pieces of a split item: a warp for two rows, lanes the dimensions, four pieces' loads together; grid (CTAs of the attention kernel, R / 16)
// 7 us where every item is split, most of it the launch and one chain of loads
template <int HD> __global__ void __launch_bounds__(256) pages_join_kernel(const __grid_constant__ KqAttnArgs a) {
    KQ_PDL_ENTER();
    const int4 meta = a.meta[2 * blockIdx.x], seq = a.meta[2 * blockIdx.x + 1];
    if (meta.x == 0) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r0 = blockIdx.y * 16 + 2 * warp;
    if ((meta.z * R + r0) / a.G >= seq.y) return;
    constexpr int N = HD / 64;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    float2 o[2][N];
#pragma unroll
    for (int k = 0; k < 2; k++)
#pragma unroll
        for (int u = 0; u < N; u++) o[k][u] = make_float2(0.f, 0.f);
    for (int i0 = 0; i0 < meta.x; i0 += 4) {
        float2 v[2][4][N];
        float4 ml[4]; // of both rows
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int i = i0 + j;
            ml[j] = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
            const float *p = a.part + (int64_t)(2 * (blockIdx.x + i) + (i == 0 ? 1 : 0)) * R * (HD + 2); // piece 0 is slot 2 b + 1, piece i slot 2 (b + i)
            if (i < meta.x) ml[j] = *reinterpret_cast<const float4 *>(p + R * HD + 2 * r0);
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int u = 0; u < N; u++) v[k][j][u] = i < meta.x ? *reinterpret_cast<const float2 *>(p + (r0 + k) * HD + 2 * (lane + 32 * u)) : make_float2(0.f, 0.f);
        }
#pragma unroll
        for (int k = 0; k < 2; k++) {
            float mn = m[k];
#pragma unroll
            for (int j = 0; j < 4; j++) mn = fmaxf(mn, k ? ml[j].z : ml[j].x);
            const float sub = mn == -INFINITY ? 0.f : mn, f0 = kq_ex2(m[k] - sub);
            l[k] *= f0;
#pragma unroll
            for (int u = 0; u < N; u++) o[k][u].x *= f0, o[k][u].y *= f0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float f = kq_ex2((k ? ml[j].z : ml[j].x) - sub);
                l[k] += f * (k ? ml[j].w : ml[j].y);
#pragma unroll
                for (int u = 0; u < N; u++) o[k][u].x += f * v[k][j][u].x, o[k][u].y += f * v[k][j][u].y;
            }
            m[k] = mn;
        }
    }
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int rr = meta.z * R + r0 + k, tok = rr / a.G;
        if (tok >= seq.y) continue;
        const float inv = l[k] == 0.f ? 0.f : 1.f / l[k];
#pragma unroll
        for (int u = 0; u < N; u++)
            kq_st2_type(a.type, a.out, (int64_t)(seq.x + tok) * a.out_stride + (int64_t)(meta.y * a.G + rr - tok * a.G) * HD + 2 * (lane + 32 * u), o[k][u].x * inv, o[k][u].y * inv);
    }
}

template <int HD, bool F8, typename T> b200_status launch(const KqAttnArgs &a, const CUtensorMap &k, const CUtensorMap &v, int box_rows, int ctas, cudaStream_t st) {
    constexpr int smem = Layout<HD, F8, std::is_same<T, __nv_bfloat16>::value ? 1 : 2>::TOTAL;
    static bool attr[64];
    int dev = 0;
    KQ_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !attr[dev]) {
        KQ_CUDA(cudaFuncSetAttribute(pages_prompt_kernel<HD, F8, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        if (dev >= 0 && dev < 64) attr[dev] = true;
    }
    kq_launch(pages_prompt_kernel<HD, F8, T>, ctas, F8 ? 512 : 384, smem, st, a, k, v, box_rows);
    KQ_COUNT_LAUNCH();
    KQ_LAUNCH_CHECK();
    return B200_OK;
}
template <int HD, bool F8> b200_status launch(const KqAttnArgs &a, const CUtensorMap &k, const CUtensorMap &v, int box_rows, int ctas, cudaStream_t st) {
    if (a.type == B200_TYPE_F32) return launch<HD, F8, float>(a, k, v, box_rows, ctas, st);
    return a.type == B200_TYPE_F16 ? launch<HD, F8, __half>(a, k, v, box_rows, ctas, st) : launch<HD, F8, __nv_bfloat16>(a, k, v, box_rows, ctas, st);
}

constexpr size_t META_BYTES = 8192;

} // namespace

int kq_pages_error_fetch() {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_pages_error, sizeof(int)) != cudaSuccess) return -1;
    if (v) cudaMemcpyToSymbol(g_pages_error, &zero, sizeof(int));
    return v;
}

size_t kq_pages_prompt_scratch(int hd) { return META_BYTES + (size_t)kq_sm_count() * R * (2 * (hd + 2) + hd + 2) * sizeof(float); } // two slots of a CTA, and what it puts aside

b200_status kq_pages_prompt(KqAttnArgs a, bool f8, int hd, uint8_t *scratch, cudaStream_t st) {
    const int ctas = kq_sm_count();
    KQ_REQUIRE((size_t)ctas * 2 * sizeof(int4) <= META_BYTES, "attention_pages: %d multiprocessors", ctas);
    a.meta = (int4 *)scratch;
    a.part = (float *)(scratch + META_BYTES);
    int box_rows = 128; // the largest power of two that divides the page
    while (a.c.page % box_rows) box_rows /= 2;
    CUtensorMap maps[2];
    memset(maps, 0, sizeof(maps));
    if (!f8)
        for (int i = 0; i < 2; i++) {
            const uint64_t dims[3] = {(uint64_t)hd, (uint64_t)a.c.n_kv * a.c.page, (uint64_t)a.c.n_pages}, strides[2] = {(uint64_t)hd * 2, (uint64_t)a.c.page_bytes};
            const uint32_t box[3] = {64, (uint32_t)box_rows, 1};
            KQ_TRY(kq_tmap_encode(&maps[i], 2, 3, i ? a.c.v : a.c.k, dims, strides, box, 1));
        }
    if (hd == 128) KQ_TRY(f8 ? (launch<128, true>(a, maps[0], maps[1], box_rows, ctas, st)) : (launch<128, false>(a, maps[0], maps[1], box_rows, ctas, st)));
    else KQ_TRY(f8 ? (launch<64, true>(a, maps[0], maps[1], box_rows, ctas, st)) : (launch<64, false>(a, maps[0], maps[1], box_rows, ctas, st)));
    kq_launch(hd == 128 ? pages_join_kernel<128> : pages_join_kernel<64>, dim3((unsigned)ctas, R / 16), 256, 0, st, a);
    KQ_COUNT_LAUNCH();
    KQ_LAUNCH_CHECK();
    return B200_OK;
}
