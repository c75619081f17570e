// vxc_kv8_attn_many.cu — attention over the paged 8-bit KV cache for many
// queries per kv head (prompt pieces, wide verify steps) on tcgen05
// (reference src/model.c:299-338, over its fp32 cache).
//
// CTA = (tile of 128, 64 or 32 queries of one request and kv head) x one split
// of its tokens; queries are row * G + head, so a tile is 128 / G consecutive
// rows and its causal bound is tight.  Tokens go by in tiles of 128:
//   S = Q K^T    two products per step of 16, Q_hi and Q_lo (from TMEM)
//   P            softmax weights in place of S in TMEM, hi and lo fp16
//   O = P V      two products per step
// Codes are exact in fp16; Q rows (scaled by a power of two) and weights are
// split into two fp16 parts, 22 bits together, so products are fp32-exact in
// effect.  Each tile's O starts from zero and is added to fp32 registers: the
// tensor core's own sums lose up to an ulp a step and stay 16 steps long, and
// no rescaling of TMEM is needed.
// Bound: tensor work, 2 x 2 x 128 x 128 x head_dim multiply-adds per tile
// (2048 cycles at head dim 128), and shared memory, which K and V pass as bytes
// (in and out), as fp16 (in) and as operands: as much time again.  (Q from
// shared memory added half of that: hence in TMEM.)
//
// Roles (640 threads, one CTA per SM):
//   warps 0-7    loaders: convert raw rows to fp16 core matrices
//   warps 8-15   softmax, two threads per query: warps 8-11 have tokens 0-63 of
//                a tile and the first half of the output columns, warps 12-15
//                the others; they exchange their maxima through shared memory.
//                Weights of tile j first, then O of tile j - 1 is added, so its
//                product runs beside them.  In tiles of 64 or 32 queries the
//                queries stand in 2 or 4 copies, which share a tile's tokens
//   warp 16      issues S of tile j + 2; warp 17 issues P V of tile j
//   warp 18      block table and scales of the coming tiles, four at a time
//   warp 19      bulk copies of raw rows, a span of 16 tokens each, MN_AHEAD
//                pieces (K or V of a tile) ahead
// TMEM: two buffers of 128 columns for S / P, 128 for O, 128 for Q.
// K and V tiles have two slots each.  K as [head dim chunk][token] x 16 bytes
// is K-major, V in the same layout is MN-major; chunks are 2064 bytes apart, so
// the loaders' 16-byte stores fall into different banks.  Queries come and
// outputs go as whole rows, through V's slots before and after their use.
//
// Measured (heads of 128): 4096 rows behind 12288 tokens, 64 heads over 8,
// 3.43 ms: 561 Tflop/s of attention, 1.12 Pflop/s of fp16 products, 0.67 of a
// library's bf16 product.  8 prompts of up to 512 rows, 32 heads, 96 us; 32
// requests of 7 rows behind up to 4096 tokens, 64 heads over 8, 84 us one call
// after the other (89 to 91 us among other work).  Bound:
// a tile takes 3700 cycles, of which 2048 are products.  The softmax warps'
// chain is as long: waiting for and reading S 900, maxima 400, weights 1800 (64
// of each thread's exponentials and conversions share a unit of 16 lanes), O
// 450, and the next product starts behind it (one O fits TMEM at head dim 128).  A CTA costs
// 11 us besides, mostly latencies one after the other: lookups, queries, first
// tile, last product, output; hence short requests' distance from their floor.
// Slower: one thread per query (-9 %); each half of the softmax warps on a tile
// of its own (-5 to -10 %); persistent CTAs over a list of tiles (-20 %); 128
// loader threads; queries as operands from shared memory; O added beside or
// before the weights (-15 to -40 %: TMEM reads queue behind its stores); loaders
// with cp.async of their own (they were the longest chain, 3750 cycles a tile);
// arrivals of threads instead of warps.
// Every wait is bounded (VXC_WAIT_NS); on expiry the error word is set, every
// role leaves its loop, and TMEM is freed after the issued work has ended.
#include "vxc_kv8_attn.cuh"

#define MN_LOADERS 256         // warps 0-7
#define MN_THREADS (MN_LOADERS + 256 + 128)
#define MN_CHUNK 2064          // bytes between 8-column chunks of a 128-row fp16 tile
#define MN_PAGES 8             // tiles whose blocks and scales are held
#define MN_AHEAD 4             // K or V pieces of raw bytes in flight

template <int HD>
struct MnSmem {
    static constexpr int TILE = HD / 8 * MN_CHUNK;          // one fp16 tile of 128 rows
    static constexpr int PIECE = 128 * HD;                  // its bytes as they come from the cache
    // V's tiles, before them the queries and after them the outputs: 128 rows of HD + 4 floats
    static constexpr int QO = 128 * (HD + 4) * 4, VQO = 2 * TILE > QO ? 2 * TILE : QO;
    static constexpr int K = 0, RAW = 2 * TILE, V = RAW + MN_AHEAD * PIECE, BYTES = V + VQO;
};

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}

// Two floats at once.
__device__ __forceinline__ uint64_t f2(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void unf2(uint64_t v, float &x, float &y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]),
                 "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

// mbar_wait behind a first look without a suspend hint: most phases are complete when asked for.
__device__ __forceinline__ bool mn_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag, unsigned int *err,
                                        unsigned int code) {
    return mbar_try(bar, parity) || mbar_wait(bar, parity, abort_flag, err, code);
}

// The factor of a group's scores, kept above 0: a masked score (-inf) times it is -inf, never NaN.
// (Where it would be less, a score is below 1e-25 either way: the weight is the same.)
__device__ __forceinline__ float mn_factor(float x) { return fmaxf(x, 1e-37f); }

// The softmax warps only.
__device__ __forceinline__ void mn_group_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// One lane of the (whole) warp, the same one each time: products and their commits are one thread's.  (With
// `lane == 0` instead the compiler does not see that one thread runs, and each product took 100 cycles to issue.)
__device__ __forceinline__ bool mn_elect() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}

// Every warp, at the end of its role.  Registers go back to what the block was launched with only behind
// this: a warp that is done early (one has nothing to do at all) would otherwise take back registers that a
// softmax warp has not got yet, and that warp would wait for them for ever.
__device__ __forceinline__ void mn_roles_done() { asm volatile("bar.sync 2, %0;" ::"n"(MN_THREADS) : "memory"); }

template <int TYPE, int HD, int TQ>
__global__ void __launch_bounds__(MN_THREADS, 1) k_kv8_attn_many(const Kv8AttnArgs a) {
    using M = MnSmem<HD>;
    extern __shared__ __align__(128) unsigned char sm[];
    __shared__ __align__(8) uint64_t bars[18 + 3 * MN_PAGES + MN_AHEAD];
    __shared__ long long page_at[MN_PAGES][8];     // byte offset of a 16-token group in the cache; -1 none, -2 bad block
    __shared__ __align__(16) float page_ks[MN_PAGES][8], page_vs[MN_PAGES][8], page_lv[MN_PAGES][8];
    __shared__ float2 red[2][2][128];              // [tile parity][half][query]: maxima of half a tile
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    __shared__ struct {
        const int *table;
        int q0, nq, row0, pos, kvlen, ns, SL;   // nq 0: no work
    } item;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int KH = a.kv.n_kv_heads, G = a.H / KH, bs = a.kv.block_size;
    // heads and splits of a tile stand together: tiles begin in their order, over the whole grid
    const int tiles = (int)gridDim.x / (KH * a.S), tile = (int)blockIdx.x / (KH * a.S);
    const int kvh = ((int)blockIdx.x - tile * KH * a.S) / a.S, split = ((int)blockIdx.x - tile * KH * a.S) % a.S;
    const uint32_t bar0 = smem_u32(bars);
    // warps arrive, not threads: 32 arrivals are 32 atomics on one word
    auto kfull = [&](int s) { return bar0 + 8u * s; };             // K tile stored (loader warps)
    auto vfull = [&](int s) { return bar0 + 8u * (2 + s); };
    auto rfull = [&](int s) { return bar0 + 8u * (4 + s); };       // raw piece landed (bytes)
    auto sfull = [&](int b) { return bar0 + 8u * (8 + b); };       // S product of a tile in buffer b done: its K slot is free
    auto pfull = [&](int b) { return bar0 + 8u * (10 + b); };      // its weights stored (softmax warps)
    auto ofull = [&](int b) { return bar0 + 8u * (12 + b); };      // its P V product done: its V slot is free
    const uint32_t oempty = bar0 + 8u * 14, qfull = bar0 + 8u * 15;   // O read; queries stored (softmax warps)
    auto gfull = [&](int s) { return bar0 + 8u * (18 + s); };      // blocks of a tile known; its scales
    auto gscale = [&](int s) { return bar0 + 8u * (18 + 2 * MN_PAGES + MN_AHEAD + s); };
    auto gempty = [&](int s) { return bar0 + 8u * (18 + MN_PAGES + s); };   // the copy warp and the softmax warps are done with them
    auto rempty = [&](int s) { return bar0 + 8u * (18 + 2 * MN_PAGES + s); };   // raw piece read (loader warps)
    static_assert(MN_AHEAD <= 4, "rfull has places 4-7");
    if (tid == 32) {
        for (int s = 0; s < 2; s++) {
            mbar_init(kfull(s), MN_LOADERS / 32), mbar_init(vfull(s), MN_LOADERS / 32);
            mbar_init(sfull(s), 1), mbar_init(pfull(s), 8), mbar_init(ofull(s), 1);
            mbar_init(bar0 + 8u * (16 + s), 1);   // an issuer's last work, after an abort
        }
        mbar_init(oempty, 8), mbar_init(qfull, 8);
        for (int s = 0; s < MN_PAGES; s++) mbar_init(gfull(s), 1), mbar_init(gscale(s), 1), mbar_init(gempty(s), 1 + 8);
        for (int s = 0; s < MN_AHEAD; s++) mbar_init(rfull(s), 1), mbar_init(rempty(s), MN_LOADERS / 32);
        abort_flag = 0;
        mbar_init_fence();
    }
    if (warp == 16) tmem_alloc(smem_u32(&tmem_slot), 512u);
    pdl_wait();
    int nth = tiles - 1 - tile;
    if (a.ranked && tid < KV8_RANKED) nth = kv8_ranked(a, tile, reinterpret_cast<int *>(sm));
    if (warp == 0) {
        // request and query tile: tiles of request r begin at floor(row0 G / TQ) + r, which leaves
        // every request as many as it needs; later tiles (longer contexts) first.  (One warp: the
        // same work by all of them took 2000 cycles more.)
        const bool one = tiles == a.n_req;   // a tile per request
        const int idx = nth;
        int r = one ? idx : 0, len = one ? 1 : a.n_req, r0, r1, pos, seq;
        do {   // 32 places a step
            const int step = (len + 31) / 32, at = lane * step, ri = r + at;
            const bool in = at < len;
            r0 = in ? kv8_row0(a, ri) : 0;
            if (step == 1) {
                r1 = in ? kv8_row0(a, ri + 1) : 0;
                pos = in ? a.pos[ri] : 0;
                seq = in && a.seq ? a.seq[ri] : ri;
            }
            const bool le = in && (one || (long long)max(r0, 0) * G / TQ + ri <= idx);
            const unsigned mask = __ballot_sync(0xffffffffu, le);
            const int k = mask ? 31 - __clz(mask) : 0;
            r += k * step;
            if (step == 1) {
                r0 = __shfl_sync(0xffffffffu, r0, k);
                r1 = __shfl_sync(0xffffffffu, r1, k);
                pos = __shfl_sync(0xffffffffu, pos, k);
                seq = __shfl_sync(0xffffffffu, seq, k);
                break;
            }
            len = min(step, len - k * step);
        } while (true);
        const Kv8Req rq = kv8_req_of(a, seq, r0, r1, pos);
        const long long tile0 = one ? idx : (long long)rq.row0 * G / TQ + r;
        if (kvh == 0 && split == 0 && lane == 0 &&
            ((rq.over && idx == tile0) || (idx == 0 && kv8_row0(a, a.n_req) > a.n_rows)))
            vxc_flag_error(a.err, VXC_DERR_BAD_BLOCK);
        const int nq = rq.T * G;
        const long long q0 = (idx - tile0) * TQ;
        int SL;
        const int ns = kv8_splits(rq.kvlen, a.sl_min, a.S, SL);
        if (lane == 0) {
            const bool work = q0 >= 0 && q0 < nq && split < ns;
            item.q0 = (int)q0, item.nq = work ? nq : 0, item.row0 = rq.row0, item.pos = rq.pos, item.kvlen = rq.kvlen;
            item.ns = ns, item.SL = SL, item.table = rq.table;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const int q0 = item.q0, nq = item.nq, row0 = item.row0, pos = item.pos, kvlen = item.kvlen, ns = item.ns;
    const int p0 = split * item.SL, p1 = min(p0 + item.SL, pos + (min(q0 + TQ, nq) - 1) / G + 1);
    const int nt = p1 > p0 ? (p1 - p0 + 127) >> 7 : 0;
    if (nq == 0) {   // nothing here
        if (warp == 16) tmem_dealloc(tmem_slot, 512u);
        return;
    }
    const uint32_t tmem = tmem_slot, t_o = tmem + 256, t_q = tmem + 384;   // Q: hi in HD / 2 columns, lo 64 columns on
    volatile int *abortp = &abort_flag;
    unsigned int *err = a.err;
    const uint32_t smb = smem_u32(sm);

    // pieces in the order K0, K1, V0, K2, V1, ..., V(nt - 1)
    const int np = 2 * nt;
    auto tile_of = [&](int i) { return i == 0 ? 0 : i == np - 1 ? nt - 1 : (i & 1) ? (i + 1) / 2 : i / 2 - 1; };
    auto is_v = [&](int i) { return i == np - 1 || (i != 0 && (i & 1) == 0); };
    // one arrival for the warp, after what all its lanes have done
    auto warp_arrive = [&](uint32_t bar) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
    };

    if (warp < MN_LOADERS / 32) {
        // ------------------------------ loaders ------------------------------
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        // 16-byte units, TPR threads a row
        constexpr int TPR = HD == 96 ? 8 : HD / 16, RP = MN_LOADERS / TPR, NP = 128 / RP;   // rows a pass, passes
        const int c = tid % TPR, tr = tid / TPR;
        const bool on = c < HD / 16;
        bool ok = true;
#pragma unroll 1
        for (int i = 0; i < np && ok; i++) {
            const int j = tile_of(i), s = j & 1, slot = i % MN_AHEAD;
            const bool isv = is_v(i);
            ok = mn_wait(rfull(slot), (i / MN_AHEAD) & 1, abortp, err, VXC_DERR_TIMEOUT_TMA);
            if (ok && j >= 2) ok = mn_wait(isv ? ofull(s) : sfull(s), ((j >> 1) - 1) & 1, abortp, err, VXC_DERR_TIMEOUT_MMA);
            if (ok && isv && j == 0) ok = mn_wait(qfull, 0, abortp, err, VXC_DERR_TIMEOUT_EPI);   // V's space held the queries
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const int live = kvlen - (p0 + 128 * j);   // rows behind the request's last token count as zeros
            unsigned char *dst = sm + (isv ? M::V : M::K) + s * M::TILE + 2 * c * MN_CHUNK + tr * 16;
            const unsigned char *src = sm + M::RAW + slot * M::PIECE + tr * HD + c * 16;
            // of its two chunks a thread stores the second one first if c & 4: eight threads of a row
            // then store into different banks
            const bool swap = (c & 4) != 0;
            unsigned char *d0 = dst + (swap ? MN_CHUNK : 0), *d1 = dst + (swap ? 0 : MN_CHUNK);
            if (on) {
#pragma unroll
                for (int k = 0; k < NP; k++) {
                    uint4 w = *reinterpret_cast<const uint4 *>(src + k * (RP * HD));
                    if (live < 128 && k * RP + tr >= live) w = make_uint4(0, 0, 0, 0);
                    uint4 h0, h1;
                    codes_h2<TYPE>(swap ? w.z : w.x, h0.x, h0.y);
                    codes_h2<TYPE>(swap ? w.w : w.y, h0.z, h0.w);
                    codes_h2<TYPE>(swap ? w.x : w.z, h1.x, h1.y);
                    codes_h2<TYPE>(swap ? w.y : w.w, h1.z, h1.w);
                    *reinterpret_cast<uint4 *>(d0 + k * RP * 16) = h0;
                    *reinterpret_cast<uint4 *>(d1 + k * RP * 16) = h1;
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(isv ? vfull(s) : kfull(s));
                mbar_arrive(rempty(slot));
            }
        }
        __syncwarp();
        mn_roles_done();
        asm volatile("setmaxnreg.inc.sync.aligned.u32 96;");
    } else if (warp < MN_LOADERS / 32 + 8) {
        // ------------------------------ softmax ------------------------------
        constexpr int HC = HD / 2;   // elements of a query, columns of O per thread
        // TQ < 128: the tile's queries stand in 128 / TQ parts of its rows, and each part weighs its own
        // tokens of a tile (the others' weights are 0 there): NG groups of 16 tokens per thread
        constexpr int NP = 128 / TQ, NG = 4 / NP;
        const int half = (warp >> 2) - MN_LOADERS / 128, row = tid & 127, part = row / TQ, qrow = row % TQ;
        const uint32_t tl = (uint32_t)((warp & 3) * 32) << 16;
        const int q = q0 + qrow;
        // Global rows are read and written whole, LPR lanes a row (a lane per row would touch 32 lines an
        // instruction), and change hands in shared memory
        constexpr int LPR = HD == 96 ? 32 : HD / 4, RPW = 32 / LPR, XS = HD + 4;
        constexpr int RPS = 8 * RPW;   // rows a step
        const int srow = (warp - MN_LOADERS / 32) * RPW + lane / LPR, scol = 4 * (lane % LPR);   // rows srow + RPS i
        const bool son = scol < HD;
        // query srow's row and head, and how far RPS queries are
        const int t_at = (q0 + srow) / G, g_at = q0 + srow - t_at * G, t_by = RPS / G, g_by = RPS - t_by * G;
        float *xs = reinterpret_cast<float *>(sm + M::V);
        {   // queries on their way (before the wait for registers)
            int g = g_at;
            const float *src = a.q + (size_t)(row0 + t_at) * a.ldq + (size_t)(kvh * G + g) * HD + scol;
            const long long step = (long long)t_by * a.ldq + (long long)g_by * HD, wrap = a.ldq - (long long)G * HD;
#pragma unroll
            for (int i = 0; i < TQ / RPS; i++) {
                const int rw = srow + RPS * i;
                const bool have = rw < nq - q0;
                if (son) cp_async_zfill<16>(smem_u32(xs + rw * XS + scol), have ? src : a.q, have);
                src += step;
                g += g_by;
                if (g >= G) g -= G, src += wrap;
            }
            cp_commit();
        }
        asm volatile("setmaxnreg.inc.sync.aligned.u32 160;");
        float f;   // factor of the query's scores
        {
            // half a query into TMEM
            cp_wait<0>();
            mn_group_sync();
            float4 v[HC / 4];
            float mx = 0.0f;
#pragma unroll
            for (int c = 0; c < HC / 4; c++) {
                v[c] = *reinterpret_cast<const float4 *>(xs + qrow * XS + half * HC + 4 * c);
                mx = fmaxf(mx, fmaxf(fmaxf(fabsf(v[c].x), fabsf(v[c].y)), fmaxf(fabsf(v[c].z), fabsf(v[c].w))));
            }
            red[1][half][row].x = mx;
            mn_group_sync();
            mx = fmaxf(mx, red[1][half ^ 1][row].x);
            // the row's largest element into [2^13, 2^14); a negative scale goes into the queries, since
            // the maxima are taken before the factor is applied
            const int ex = min(max((int)(__float_as_uint(mx) >> 23), 14), 253);
            const float up = copysignf(__uint_as_float((uint32_t)(267 - ex) << 23), a.scale);
            f = fabsf(a.scale) * 1.4426950408889634f * __uint_as_float((uint32_t)(ex - 13) << 23);
#pragma unroll
            for (int c = 0; c < HC / 16; c++) {
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float4 x = v[4 * c + i];
                    hi[2 * i] = split_h2(x.x * up, x.y * up, lo[2 * i]);
                    hi[2 * i + 1] = split_h2(x.z * up, x.w * up, lo[2 * i + 1]);
                }
                tmem_st8(t_q + tl + half * (HC / 2) + 8 * c, hi);
                tmem_st8(t_q + tl + 64 + half * (HC / 2) + 8 * c, lo);
            }
            tmem_wait_st();
            tc_fence_before();
            warp_arrive(qfull);
        }
        float m = -INFINITY, mv = -INFINITY, l = 0.0f;
        float acc[HC];
#pragma unroll
        for (int d = 0; d < HC; d++) acc[d] = 0.0f;
        // (places without a query: as the last one, so that they do not cost their warp the masks)
        const int lim = pos + min(q, nq - 1) / G;
        // adds O of tile j to the registers
        auto drain = [&](int j) -> bool {
            const bool there = mn_wait(ofull(j & 1), (j >> 1) & 1, abortp, err, VXC_DERR_TIMEOUT_MMA);
            if (!__all_sync(0xffffffffu, there)) return false;
            tc_fence_after();
            uint32_t v[HC];
#pragma unroll
            for (int c = 0; c < HC / 16; c++) tmem_ld16(t_o + tl + half * HC + 16 * c, v + 16 * c);
            tmem_wait_ld();
            tmem_pin<HC>(v);
#pragma unroll
            for (int d = 0; d < HC; d += 2)
                unf2(add2(f2(acc[d], acc[d + 1]), f2(__uint_as_float(v[d]), __uint_as_float(v[d + 1]))), acc[d], acc[d + 1]);
            tc_fence_before();
            warp_arrive(oempty);
            return true;
        };
        bool ok = true;
#pragma unroll 1
        for (int j = 0; j < nt; j++) {
            const int e = j % MN_PAGES, b = j & 1;
            const uint32_t t_s = tmem + tl + 128 * b + 64 * half, t_g = t_s + 16 * NG * part;
            const int g0 = 4 * half + NG * part;   // the thread's first group of 16 tokens
            // (S is there, so the loaders have seen the tile's blocks and scales, and so does this thread)
            ok = ok && mn_wait(sfull(b), (j >> 1) & 1, abortp, err, VXC_DERR_TIMEOUT_MMA);
            // (after a failed wait the scores are garbage; every warp leaves at the barrier below)
            __syncwarp();
            tc_fence_after();
            uint32_t v[16 * NG];
            float mx = -INFINITY, mxv = -INFINITY, shrink = 1.0f;
            if constexpr (NG == 1) {
                tmem_ld16(t_g, v);
            } else {
                tmem_ld32(t_g, v);
                if constexpr (NG == 4) tmem_ld32(t_g + 32, v + 32);
            }
            const int t0 = p0 + 128 * j + 16 * g0;
            float fk[NG];
#pragma unroll
            for (int c = 0; c < NG; c++) fk[c] = mn_factor(f * page_ks[e][g0 + c]);
            // bit c: group c of 16 tokens lies in a block outside the cache
            const uint32_t bad = __ballot_sync(0xffffffffu, lane < NG && page_at[e][g0 + (lane & (NG - 1))] == -2);
            const bool whole = __all_sync(0xffffffffu, lim >= t0 + 16 * NG - 1) && bad == 0;
            tmem_wait_ld();
            tmem_pin<16 * NG>(v);
            if (NP > 1) {
                const uint32_t none[16] = {};
#pragma unroll
                for (int g = 0; g < 4; g++)
                    if (g / NG != part) tmem_st16(t_s + 16 * g, none);
            }
            if (!whole) {
#pragma unroll
                for (int c = 0; c < NG; c++) {   // visible tokens of group c: the low bits of a mask
                    const int n = lim - (t0 + 16 * c) + 1;
                    const uint32_t mk = ((bad >> c) & 1u) || n <= 0 ? 0u : n >= 16 ? 0xFFFFu : (1u << n) - 1u;
#pragma unroll
                    for (int k = 0; k < 16; k++) v[16 * c + k] = (mk >> k) & 1u ? v[16 * c + k] : 0xFF800000u;   // -inf
                }
            }
#pragma unroll
            for (int c = 0; c < NG; c++) {
                float x = __uint_as_float(v[16 * c]);
#pragma unroll
                for (int k = 1; k < 16; k++) x = fmaxf(x, __uint_as_float(v[16 * c + k]));
                x *= fk[c];
                mx = fmaxf(mx, x);
                mxv = fmaxf(mxv, x + page_lv[e][g0 + c]);
            }
            red[b][half][row] = make_float2(mx, mxv);
            ok = bar_and(1, 256, ok);   // the softmax warps go on together or not at all
            if (!ok) break;
#pragma unroll
            for (int i = 1; i < 2 * NP; i++) {   // the query's other threads
                const float2 o = red[b][half ^ (i & 1)][qrow + TQ * ((part + (i >> 1)) % NP)];
                mx = fmaxf(mx, o.x);
                mxv = fmaxf(mxv, o.y);
            }
            if (mx > m + KV8_LAG || (m == -INFINITY && mx > m)) {
                l *= ex2(m - mx);   // 0 at first
                m = mx;
            }
            const float least = m - KV8_FLOOR;
            mxv = fmaxf(mxv, least);
            if (mxv > mv + KV8_LAG || least > mv) {
                shrink = ex2(mv - mxv);
                mv = mxv;
            }
            float mref = m == -INFINITY ? 0.0f : m;
            float cv = ex2(fminf(mref - mv + KV8_HEAD, KV8_FLOOR + KV8_HEAD));   // (no token yet: mv is -inf)
            float vmax = page_vs[e][g0];
#pragma unroll
            for (int c = 1; c < NG; c++) vmax = fmaxf(vmax, page_vs[e][g0 + c]);
            const float unit = kv8_unit(vmax, cv, mref);
            const uint64_t nm = f2(-mref, -mref), minus = f2(-1.0f, -1.0f);
            uint64_t sum = f2(0.0f, 0.0f);
#pragma unroll
            for (int c = 0; c < NG; c++) {
                // (read again: registers are what is short here)
                const float fg = mn_factor(f * page_ks[e][g0 + c]), cw = kv8_factor(page_vs[e][g0 + c], cv);
                const uint64_t fkc = f2(fg, fg), cw2 = f2(cw, cw);
                uint32_t w[16];
#pragma unroll
                for (int k = 0; k < 16; k += 2) {
                    float x, y;
                    unf2(fma2(f2(__uint_as_float(v[16 * c + k]), __uint_as_float(v[16 * c + k + 1])), fkc, nm), x, y);
                    x = ex2(x);
                    y = ex2(y);
                    const uint64_t p = f2(x, y);
                    sum = add2(sum, p);
                    float wx, wy;
                    const uint64_t wt = mul2(p, cw2);
                    unf2(wt, wx, wy);
                    const __half2 h = __floats2half2_rn(wx, wy);
                    const float2 hf = __half22float2(h);
                    unf2(fma2(f2(hf.x, hf.y), minus, wt), wx, wy);
                    const __half2 lo = __floats2half2_rn(wx, wy);
                    w[k / 2] = *reinterpret_cast<const uint32_t *>(&h);
                    w[8 + k / 2] = *reinterpret_cast<const uint32_t *>(&lo);
                }
                // hi in columns 0-7 of the group's 16, lo in 8-15
                tmem_st16(t_g + 16 * c, w);
            }
            {
                float x, y;
                unf2(sum, x, y);
                l = fmaf(x + y, unit, l);
            }
            tmem_wait_st();
            tc_fence_before();
            warp_arrive(pfull(b));
            if (lane == 0) {
                mbar_arrive(gempty(e));
            }
            if (j > 0) ok = drain(j - 1);
            if (__any_sync(0xffffffffu, shrink != 1.0f)) {
#pragma unroll
                for (int d = 0; d < HC; d++) acc[d] *= shrink;
            }
        }
        if (ok && nt > 0) ok = drain(nt - 1);
        red[0][half][row].x = l;
        ok = bar_and(1, 256, ok);
        if (ok) {
            float L = 0.0f;
#pragma unroll
            for (int i = 0; i < NP; i++) L += red[0][0][qrow + TQ * i].x + red[0][1][qrow + TQ * i].x;
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;   // no token: 0; NaN stays
            const float back = mv == -INFINITY ? 0.0f : ex2(mv - m - KV8_HEAD);
            // (every product has ended: V's space is free)
#pragma unroll
            for (int d = 0; d < HC; d += 4)
                *reinterpret_cast<float4 *>(xs + row * XS + half * HC + d) =
                    make_float4(acc[d] * inv * back, acc[d + 1] * inv * back, acc[d + 2] * inv * back, acc[d + 3] * inv * back);
            if (ns > 1 && half == 0 && part == 0 && q < nq) {
                const int t = q / G, h = kvh * G + q - t * G;
                *reinterpret_cast<float2 *>(a.part + (((size_t)(row0 + t) * a.H + h) * a.S + split) * (HD + 4)) = make_float2(m, L);
            }
            if (NP == 1) {   // each thread sends its half row
                fence_proxy_async();
                if (q < nq) {
                    const int t = q / G, h = kvh * G + q - t * G;
                    float *to = (ns > 1 ? a.part + (((size_t)(row0 + t) * a.H + h) * a.S + split) * (HD + 4) + 4
                                        : a.out + (size_t)(row0 + t) * a.ldo + (size_t)h * HD) + half * HC;
                    bulk_s2g(to, smem_u32(xs + row * XS + half * HC), HC * 4);
                }
            } else {   // the parts' sum
                mn_group_sync();
                int g = g_at;
                const size_t hw = ns > 1 ? (size_t)a.S * (HD + 4) : HD;   // a head's floats, a row's
                const long long ld = ns > 1 ? (long long)a.H * hw : a.ldo;
                float *dst = (ns > 1 ? a.part + (size_t)split * (HD + 4) + 4 : a.out) + (size_t)(row0 + t_at) * ld +
                             (size_t)(kvh * G + g) * hw + scol;
                const long long step = t_by * ld + (long long)(g_by * hw), wrap = ld - (long long)(G * hw);
#pragma unroll
                for (int i = 0; i < TQ / RPS; i++) {
                    const int rw = srow + RPS * i;
                    if (son && rw < nq - q0) {
                        float4 x = *reinterpret_cast<const float4 *>(xs + rw * XS + scol);
#pragma unroll
                        for (int k = 1; k < NP; k++) {
                            const float4 y = *reinterpret_cast<const float4 *>(xs + (rw + TQ * k) * XS + scol);
                            x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
                        }
                        *reinterpret_cast<float4 *>(dst) = x;
                    }
                    dst += step;
                    g += g_by;
                    if (g >= G) g -= G, dst += wrap;
                }
            }
        }
        asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
        mn_roles_done();
    } else {
        int blk0 = -1;   // the page warp's first lookup, on its way early: the first tile waits for it
        if (warp == 18 && p0 + 16 * lane < kvlen && (lane >> 3) < nt) blk0 = item.table[(p0 + 16 * lane) / bs];
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        if (warp == 16) {
            // ------------------------------ S = Q K^T ------------------------------
            const uint32_t idesc = (1u << 4) | ((uint32_t)(128 >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
            bool ok = nt > 0 && mbar_wait_warp(qfull, 0, abortp, err, VXC_DERR_TIMEOUT_EPI);
#pragma unroll 1
            for (int j = 0; j < nt && ok; j++) {
                const int s = j & 1;
                ok = mbar_wait_warp(kfull(s), (j >> 1) & 1, abortp, err, VXC_DERR_TIMEOUT_TMA);
                // the buffer's weights (tile j - 2) have been multiplied
                if (ok && j >= 2) ok = mbar_wait_warp(ofull(s), ((j >> 1) - 1) & 1, abortp, err, VXC_DERR_TIMEOUT_MMA);
                // (the softmax warps read the scales once S is there)
                ok = ok && mbar_wait_warp(gscale(j % MN_PAGES), (j / MN_PAGES) & 1, abortp, err, VXC_DERR_TIMEOUT_EPI);
                if (!ok) break;
                tc_fence_after();
                const uint64_t kd = sdesc(smb + M::K + s * M::TILE, MN_CHUNK, 128);
                const uint32_t d = tmem + 128 * s;
                if (mn_elect()) {
#pragma unroll
                    for (int k = 0; k < HD / 16; k++) {
                        const uint64_t bd = kd + (uint64_t)((k * 2 * MN_CHUNK) >> 4);
                        mma_f16_ts(d, t_q + 8 * k, bd, idesc, k != 0);
                        mma_f16_ts(d, t_q + 64 + 8 * k, bd, idesc, 1u);
                    }
                    mma_commit(sfull(s));
                }
                __syncwarp();
            }
        } else if (warp == 17) {
            // ------------------------------ O = P V ------------------------------
            // V is MN-major (bit 16): 8-column chunks MN_CHUNK apart, groups of 8 tokens 128 bytes apart
            const uint32_t idesc = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
            bool ok = true;
#pragma unroll 1
            for (int j = 0; j < nt && ok; j++) {
                const int s = j & 1;
                ok = mbar_wait_warp(vfull(s), (j >> 1) & 1, abortp, err, VXC_DERR_TIMEOUT_TMA);
                ok = ok && mbar_wait_warp(pfull(s), (j >> 1) & 1, abortp, err, VXC_DERR_TIMEOUT_MMA);
                if (ok && j >= 1) ok = mbar_wait_warp(oempty, (j - 1) & 1, abortp, err, VXC_DERR_TIMEOUT_MMA);
                if (!ok) break;
                tc_fence_after();
                const uint64_t vd = sdesc(smb + M::V + s * M::TILE, 128, MN_CHUNK);
                const uint32_t p = tmem + 128 * s;
                if (mn_elect()) {
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        const uint64_t bd = vd + (uint64_t)((k * 256) >> 4);
                        mma_f16_ts(t_o, p + 16 * k, bd, idesc, k != 0);
                        mma_f16_ts(t_o, p + 16 * k + 8, bd, idesc, 1u);
                    }
                    mma_commit(ofull(s));
                }
                __syncwarp();
            }
        } else if (warp == 18) {
            // ------------------------------ blocks and scales ------------------------------
            // lane = (tile of four, group of 16 tokens)
            bool ok = true;
#pragma unroll 1
            for (int t = 0; t < nt && ok; t += 4) {
                const int p = p0 + 128 * t + 16 * lane;
                long long at = -1;
                float ks = 0.0f, vs = 0.0f;
                if (p < kvlen && t + (lane >> 3) < nt) {
                    const int blk = t == 0 ? blk0 : item.table[p / bs];
                    if (blk >= 0 && blk < a.kv.n_blocks) {
                        const size_t bh = (size_t)blk * KH + kvh;
                        at = (long long)((bh * bs + p % bs) * HD);
                        ks = a.kv.k_scale[bh];
                        vs = a.kv.v_scale[bh];
                    } else {
                        at = -2;
                        vxc_flag_error(err, VXC_DERR_BAD_BLOCK);
                    }
                }
                for (int k = 0; k < 4 && t + k < nt; k++) {
                    const int j = t + k, e = j % MN_PAGES;
                    if (j >= MN_PAGES) ok = mn_wait(gempty(e), ((j / MN_PAGES) - 1) & 1, abortp, err, VXC_DERR_TIMEOUT_EPI);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    if (lane >> 3 == k) page_at[e][lane & 7] = at;
                    warp_arrive(gfull(e));
                }
                const float lv = lg2(vs);
                for (int k = 0; k < 4 && t + k < nt && ok; k++) {
                    const int e = (t + k) % MN_PAGES;
                    if (lane >> 3 == k) {
                        page_ks[e][lane & 7] = ks;
                        page_vs[e][lane & 7] = vs;
                        page_lv[e][lane & 7] = lv;
                    }
                    warp_arrive(gscale(e));
                }
            }
        } else if (warp == 19) {
            // ------------------------------ copies ------------------------------
            // a group of 16 tokens is one span of its block: lane = group; groups without a block are zeros
            bool ok = true;
            int i = 0;
#pragma unroll 1
            for (; i < np; i++) {
                const int j = tile_of(i), e = j % MN_PAGES, slot = i % MN_AHEAD;
                const bool isv = is_v(i);
                ok = mn_wait(gfull(e), (j / MN_PAGES) & 1, abortp, err, VXC_DERR_TIMEOUT_TMA);
                if (ok && i >= MN_AHEAD) ok = mn_wait(rempty(slot), ((i / MN_AHEAD) - 1) & 1, abortp, err, VXC_DERR_TIMEOUT_MMA);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const long long at = lane < 8 ? page_at[e][lane] : -1;
                const unsigned have = __ballot_sync(0xffffffffu, at >= 0), none = ~have & 0xFFu;
                unsigned char *raw = sm + M::RAW + slot * M::PIECE;
                if (none) {
                    for (int g = 0; g < 8; g++)
                        if ((none >> g) & 1u)
                            for (int u = lane; u < HD; u += 32)
                                *reinterpret_cast<uint4 *>(raw + g * 16 * HD + u * 16) = make_uint4(0, 0, 0, 0);
                    fence_proxy_async();   // the next piece in this place comes by the asynchronous proxy
                }
                __syncwarp();
                if (lane == 0) {
                    mbar_expect_tx(rfull(slot), __popc(have) * 16 * HD);
                    if (isv) mbar_arrive(gempty(e));
                }
                __syncwarp();
                if (at >= 0)
                    bulk_g2s(smem_u32(raw) + lane * 16 * HD, (const uint8_t *)(isv ? a.kv.v : a.kv.k) + at, 16 * HD, rfull(slot));
            }
            // after an abort: the pieces on their way land first (bounded)
            for (int k = i > MN_AHEAD ? i - MN_AHEAD : 0; k < i; k++) {
                const uint64_t t1 = vxc_globaltimer();
                while (!mbar_try(rfull(k % MN_AHEAD), (k / MN_AHEAD) & 1) && vxc_globaltimer() - t1 < 100000000ull) {}
            }
        }
        __syncwarp();
        mn_roles_done();
        asm volatile("setmaxnreg.inc.sync.aligned.u32 96;");
    }

    // ------------------------------ end ------------------------------
    if ((warp == 16 || warp == 17) && __any_sync(0xffffffffu, *abortp != 0) && mn_elect()) {
        // an aborted issuer's products may still run: wait for them (bounded)
        const uint32_t bar = bar0 + 8u * (warp == 16 ? 16 : 17);
        mma_commit(bar);
        const uint64_t t1 = vxc_globaltimer();
        while (!mbar_try(bar, 0) && vxc_globaltimer() - t1 < 100000000ull) {}
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 16) tmem_dealloc(tmem, 512u);
}

typedef void (*many_kernel_t)(const Kv8AttnArgs);
template <int TYPE, int HD>
static many_kernel_t many_kernel(int tile_q) {
    return tile_q == 32   ? k_kv8_attn_many<TYPE, HD, 32>
           : tile_q == 64 ? k_kv8_attn_many<TYPE, HD, 64>
                          : k_kv8_attn_many<TYPE, HD, 128>;
}

template <int TYPE>
static cudaError_t launch_many(const Kv8AttnArgs &a, int tile_q, int tiles, cudaStream_t st) {
    many_kernel_t f = nullptr;
    size_t smem = 0;
    switch (a.kv.head_dim) {
        case 32: f = many_kernel<TYPE, 32>(tile_q); smem = MnSmem<32>::BYTES; break;
        case 64: f = many_kernel<TYPE, 64>(tile_q); smem = MnSmem<64>::BYTES; break;
        case 96: f = many_kernel<TYPE, 96>(tile_q); smem = MnSmem<96>::BYTES; break;
        default: f = many_kernel<TYPE, 128>(tile_q); smem = MnSmem<128>::BYTES; break;
    }
    if ((long long)tiles * a.kv.n_kv_heads * a.S > INT_MAX) return cudaErrorInvalidValue;
    // TMEM is allocated whole, at smaller head dims too, where half of it would do: one CTA per SM, so at least
    // half of the shared memory is asked for
    if (smem < 116 * 1024) smem = 116 * 1024;
    cudaError_t e = kv8_allow_smem((const void *)f, smem);
    if (e != cudaSuccess) return e;
    return kv8_launch(f, dim3((unsigned)(tiles * a.kv.n_kv_heads * a.S)), dim3(MN_THREADS), smem, st, 1, a);
}

cudaError_t kv8_attn_many(const Kv8AttnArgs &a, int tile_q, int tiles, cudaStream_t st) {
    return a.kv.type == VXC_KV8_INT8 ? launch_many<VXC_KV8_INT8>(a, tile_q, tiles, st)
                                     : launch_many<VXC_KV8_E4M3>(a, tile_q, tiles, st);
}
