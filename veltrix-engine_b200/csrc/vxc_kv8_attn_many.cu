// vxc_kv8_attn_many.cu — attention over the paged 8-bit KV cache for many
// queries per kv head (prompt pieces, wide verify steps) on tcgen05
// (reference src/model.c:299-338, over its fp32 cache).
//
// CTA = (tile of 128 queries of one request and kv head) x one split of its
// tokens; queries are row * G + head, so a tile is 128 / G consecutive rows and
// its causal bound is tight.  Tokens go by in tiles of 128:
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
// Roles (512 threads, one CTA per SM):
//   warps 0-3    loaders: cp.async 8-bit rows into slots of each thread's own
//                (MN_AHEAD pieces ahead), convert, store fp16 core matrices
//   warps 4-7 and 8-11   softmax groups A and B, thread = query: even and odd
//                tiles, each with its own S / P buffer, maxima, sum and output
//                registers
//   warp 12      issues S of tile j + 2; warp 13 issues P V of tile j
//   warp 14      block table and scales of the coming tiles
// TMEM: two buffers of 128 columns for S / P, 128 for O, 128 for Q.
// K and V tiles have two slots each.  K as [head dim chunk][token] x 16 bytes
// is K-major, V in the same layout is MN-major; chunks are 2064 bytes apart, so
// the loaders' 16-byte stores fall into different banks.
// Every wait is bounded (VXC_WAIT_NS); on expiry the error word is set, every
// role leaves its loop, and TMEM is freed after the issued work has ended.
#include "vxc_kv8_attn.cuh"

#define MN_THREADS 512
#define MN_CHUNK 2064          // bytes between 8-column chunks of a 128-row fp16 tile
#define MN_PAGES 8             // tiles whose blocks and scales are held
#define MN_AHEAD 4             // K or V pieces of raw bytes in flight

template <int HD>
struct MnSmem {
    static constexpr int TILE = HD / 8 * MN_CHUNK;          // one fp16 tile of 128 rows
    static constexpr int PIECE = 128 * (HD == 96 ? 128 : HD);   // raw bytes of one (96: as 8 units per row)
    static constexpr int K = 0, V = 2 * TILE, RAW = 4 * TILE, BYTES = RAW + MN_AHEAD * PIECE;
    static_assert(4 * TILE >= (129 * HD + 512) * 4, "the join's [HD][129] and [128][4] floats lie in the K and V slots");
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

__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]),
                 "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

// The two softmax groups only.
__device__ __forceinline__ void mn_group_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

template <int TYPE, int HD>
__global__ void __launch_bounds__(MN_THREADS, 1) k_kv8_attn_many(const Kv8AttnArgs a) {
    using M = MnSmem<HD>;
    extern __shared__ __align__(128) unsigned char sm[];
    __shared__ __align__(8) uint64_t bars[18 + 2 * MN_PAGES];
    __shared__ long long page_at[MN_PAGES][8];     // byte offset of a 16-token group in the cache; -1 none, -2 bad block
    __shared__ float page_ks[MN_PAGES][8], page_vs[MN_PAGES][8], page_lv[MN_PAGES][8];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int KH = a.kv.n_kv_heads, G = a.H / KH, bs = a.kv.block_size;
    pdl_trigger();
    pdl_wait();

    // request and query tile: tiles of request r begin at floor(row0 G / 128) + r, which leaves
    // every request as many as it needs; later tiles (longer contexts) first
    const int idx = (int)gridDim.x - 1 - (int)blockIdx.x, kvh = blockIdx.y, split = blockIdx.z;
    int r = 0;
    {
        int hi = a.n_req;
        while (hi - r > 1) {
            const int mid = (r + hi) >> 1;
            if ((long long)max(a.row0[mid], 0) * G / KV8_TILE_Q + mid <= idx) r = mid; else hi = mid;
        }
    }
    const Kv8Req rq = kv8_req(a, r);
    const long long tile0 = (long long)rq.row0 * G / KV8_TILE_Q + r;
    if (kvh == 0 && split == 0 && tid == 0 && ((rq.over && idx == tile0) || (idx == 0 && a.row0[a.n_req] > a.n_rows)))
        vxc_flag_error(a.err, VXC_DERR_BAD_BLOCK);
    const int nq = rq.T * G;
    const long long q0l = (idx - tile0) * KV8_TILE_Q;
    if (q0l < 0 || q0l >= nq) return;
    const int q0 = (int)q0l;
    int SL;
    const int ns = kv8_splits(rq.kvlen, a.sl_min, a.S, SL);
    if (split >= ns) return;
    const int p0 = split * SL, p1 = min(p0 + SL, rq.pos + (min(q0 + KV8_TILE_Q, nq) - 1) / G + 1);
    const int nt = p1 > p0 ? (p1 - p0 + 127) >> 7 : 0;

    const uint32_t bar0 = smem_u32(bars);
    auto kfull = [&](int s) { return bar0 + 8u * s; };             // K tile stored (128 loaders)
    auto kempty = [&](int s) { return bar0 + 8u * (2 + s); };      // S product read it
    auto vfull = [&](int s) { return bar0 + 8u * (4 + s); };
    auto vempty = [&](int s) { return bar0 + 8u * (6 + s); };
    auto sfull = [&](int g) { return bar0 + 8u * (8 + g); };       // S product of group g's tile done
    auto pfull = [&](int g) { return bar0 + 8u * (10 + g); };      // its weights stored (128 threads)
    auto ofull = [&](int g) { return bar0 + 8u * (12 + g); };      // its P V product done
    auto oempty = [&](int g) { return bar0 + 8u * (14 + g); };     // group g has read O
    auto gfull = [&](int s) { return bar0 + 8u * (18 + s); };      // blocks and scales of a tile (8 lanes)
    auto gempty = [&](int s) { return bar0 + 8u * (26 + s); };     // loaders (after V) and the softmax group are done with them
    if (tid == 0) {
        for (int s = 0; s < 2; s++) {
            mbar_init(kfull(s), 128), mbar_init(kempty(s), 1), mbar_init(vfull(s), 128), mbar_init(vempty(s), 1);
            mbar_init(sfull(s), 1), mbar_init(pfull(s), 128), mbar_init(ofull(s), 1), mbar_init(oempty(s), 128);
            mbar_init(bar0 + 8u * (16 + s), 1);   // an issuer's last work, after an abort
        }
        for (int s = 0; s < MN_PAGES; s++) mbar_init(gfull(s), 8), mbar_init(gempty(s), 256);
        abort_flag = 0;
        mbar_init_fence();
    }
    if (warp == 12) tmem_alloc(smem_u32(&tmem_slot), 512u);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot, t_o = tmem + 256, t_q = tmem + 384;   // Q: hi in HD / 2 columns, lo 64 columns on
    float f = 0.0f;   // softmax threads: factor of the query's scores
    if (warp >= 4 && warp < 12) {
        // queries into TMEM, thread = query, groups A and B half of the head dim each
        const int q = q0 + (tid & 127), half = (warp >> 2) - 1;
        const float4 *src = reinterpret_cast<const float4 *>(a.q + (size_t)(rq.row0 + (q < nq ? q / G : 0)) * a.ldq +
                                                             (size_t)(kvh * G + q % G) * HD);
        float mx = 0.0f;
#pragma unroll 8
        for (int i = 0; i < HD / 4; i++) {
            const float4 v = src[i];
            mx = fmaxf(mx, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
        }
        // the row's largest element into [2^13, 2^14); a negative scale goes into the queries, since
        // the maxima are taken before the factor is applied
        const int ex = min(max((int)(__float_as_uint(mx) >> 23), 14), 253);
        const float up = copysignf(__uint_as_float((uint32_t)(267 - ex) << 23), a.scale);
        f = fabsf(a.scale) * 1.4426950408889634f * __uint_as_float((uint32_t)(ex - 13) << 23);
        const uint32_t dst = t_q + ((uint32_t)((warp & 3) * 32) << 16) + half * (HD / 4);
#pragma unroll 1
        for (int c = 0; c < HD / 16; c += 2) {   // 8 columns of hi and of lo from 4 float4
            uint32_t hi[8], lo[8];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float4 v = src[half * (HD / 8) + (c / 2) * 4 + i];
                hi[2 * i] = split_h2(v.x * up, v.y * up, lo[2 * i]);
                hi[2 * i + 1] = split_h2(v.z * up, v.w * up, lo[2 * i + 1]);
            }
            tmem_st8(dst + 4 * c, hi);
            tmem_st8(dst + 64 + 4 * c, lo);
        }
        tmem_wait_st();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    volatile int *abortp = &abort_flag;
    unsigned int *err = a.err;
    const uint32_t smb = smem_u32(sm);

    if (warp < 4) {
        // ------------------------------ loaders ------------------------------
        asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        // pieces in the order K0, K1, V0, K2, V1, ..., V(nt - 1); 16-byte units, TPR threads a row
        constexpr int TPR = HD == 96 ? 8 : HD / 16, RP = 128 / TPR;
        const int c = tid % TPR, tr = tid / TPR;
        const bool on = c < HD / 16;
        const uint32_t raw = smb + M::RAW + tid * 16;
        const int np = 2 * nt;
        auto tile_of = [&](int i) { return i == 0 ? 0 : i == np - 1 ? nt - 1 : (i & 1) ? (i + 1) / 2 : i / 2 - 1; };
        auto is_v = [&](int i) { return i == np - 1 || (i != 0 && (i & 1) == 0); };
        auto load = [&](int i) -> bool {
            if (i < np) {
                const int j = tile_of(i), e = j % MN_PAGES;
                const bool isv = is_v(i);
                if (!mbar_wait(gfull(e), (j / MN_PAGES) & 1, abortp, err, VXC_DERR_TIMEOUT_TMA)) return false;
                const uint8_t *base = (const uint8_t *)(isv ? a.kv.v : a.kv.k);
                const uint8_t *src = base + (tr & 15) * HD + c * 16;
                const uint32_t dst = raw + (i % MN_AHEAD) * M::PIECE;
                const int live = rq.kvlen - (p0 + 128 * j);
                if (on) {
#pragma unroll
                    for (int k = 0; k < TPR; k++) {
                        const long long at = page_at[e][k * (RP / 16) + (tr >> 4)];
                        const bool have = at >= 0 && k * RP + tr < live;
                        cp_async_zfill<16>(dst + k * 2048, have ? src + at : base, have);
                    }
                }
                if (isv) mbar_arrive(gempty(e));
            }
            cp_commit();
            return true;
        };
        bool ok = true;
        for (int i = 0; i < MN_AHEAD && ok; i++) ok = load(i);
#pragma unroll 1
        for (int i = 0; i < np && ok; i++) {
            const int j = tile_of(i), s = j & 1;
            const bool isv = is_v(i);
            cp_wait<MN_AHEAD - 1>();
            if (j >= 2) ok = mbar_wait(isv ? vempty(s) : kempty(s), ((j >> 1) - 1) & 1, abortp, err, VXC_DERR_TIMEOUT_MMA);
            if (!ok) break;
            unsigned char *dst = sm + (isv ? M::V : M::K) + s * M::TILE + 2 * c * MN_CHUNK + tr * 16;
            const unsigned char *src = sm + M::RAW + tid * 16 + (i % MN_AHEAD) * M::PIECE;
            // of its two chunks a thread stores the second one first if c & 4: eight threads of a row
            // then store into different banks
            const bool swap = (c & 4) != 0;
            unsigned char *d0 = dst + (swap ? MN_CHUNK : 0), *d1 = dst + (swap ? 0 : MN_CHUNK);
            if (on) {
#pragma unroll
                for (int k = 0; k < TPR; k++) {
                    const uint4 w = *reinterpret_cast<const uint4 *>(src + k * 2048);
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
            mbar_arrive(isv ? vfull(s) : kfull(s));
            ok = load(i + MN_AHEAD);
        }
        cp_wait<0>();
        __syncwarp();
        asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");   // what the block was launched with, for the code behind the roles
    } else if (warp < 12) {
        // ------------------------------ softmax ------------------------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
        const int grp = (warp >> 2) - 1, row = tid & 127;
        float m = -INFINITY, mv = -INFINITY, l = 0.0f;
        float acc[HD];
#pragma unroll
        for (int d = 0; d < HD; d++) acc[d] = 0.0f;
        const uint32_t tl = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t t_s = tmem + tl + 128 * grp;
        const int q = q0 + row;
        const int lim = q < nq ? rq.pos + q / G : -1;
#pragma unroll 1
        for (int j = grp; j < nt; j += 2) {
            const int e = j % MN_PAGES;
            bool ok = mbar_wait(gfull(e), (j / MN_PAGES) & 1, abortp, err, VXC_DERR_TIMEOUT_TMA);
            ok = ok && mbar_wait(sfull(grp), (j >> 1) & 1, abortp, err, VXC_DERR_TIMEOUT_MMA);
            if (!__all_sync(0xffffffffu, ok)) break;
            tc_fence_after();
            const int t0 = p0 + 128 * j;
            // bit c: group c of 16 tokens lies in a block outside the cache
            const uint32_t bad = __ballot_sync(0xffffffffu, lane < 8 && page_at[e][lane & 7] == -2);
            const bool whole = __all_sync(0xffffffffu, lim >= t0 + 127) && bad == 0;
            // visible tokens of group c: the low bits of a mask
            auto mask = [&](int c) -> uint32_t {
                const int n = lim - (t0 + 16 * c) + 1;
                return ((bad >> c) & 1u) || n <= 0 ? 0u : n >= 16 ? 0xFFFFu : (1u << n) - 1u;
            };
            float mx = -INFINITY, mxv = -INFINITY;
#pragma unroll 1
            for (int c2 = 0; c2 < 4; c2++) {
                uint32_t v[32];
                tmem_ld32(t_s + 32 * c2, v);
                const float2 ks = *reinterpret_cast<const float2 *>(&page_ks[e][2 * c2]);
                const float2 lv = *reinterpret_cast<const float2 *>(&page_lv[e][2 * c2]);
                tmem_wait_ld();
                tmem_pin<32>(v);
                if (!whole) {
                    const uint32_t mk = mask(2 * c2) | mask(2 * c2 + 1) << 16;
#pragma unroll
                    for (int k = 0; k < 32; k++) v[k] = (mk >> k) & 1u ? v[k] : 0xFF800000u;   // -inf
                }
                float x[2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    x[h] = __uint_as_float(v[16 * h]);
#pragma unroll
                    for (int k = 1; k < 16; k++) x[h] = fmaxf(x[h], __uint_as_float(v[16 * h + k]));
                }
                // (no visible token: -inf, also where the scale is 0)
                x[0] = x[0] == -INFINITY ? x[0] : x[0] * (f * ks.x);
                x[1] = x[1] == -INFINITY ? x[1] : x[1] * (f * ks.y);
                mx = fmaxf(mx, fmaxf(x[0], x[1]));
                mxv = fmaxf(mxv, fmaxf(x[0] + lv.x, x[1] + lv.y));
            }
            if (mx > m + KV8_LAG || (m == -INFINITY && mx > m)) {
                l *= ex2(m - mx);   // 0 at first
                m = mx;
            }
            float shrink = 1.0f;
            if (mxv > mv + KV8_LAG || (mv == -INFINITY && mxv > mv)) {
                shrink = ex2(mv - mxv);
                mv = mxv;
            }
            if (__any_sync(0xffffffffu, shrink != 1.0f)) {
#pragma unroll
                for (int d = 0; d < HD; d++) acc[d] *= shrink;
            }
            const float mref = m == -INFINITY ? 0.0f : m;
            const float cv = ex2(fminf(mref - mv + KV8_HEAD, 120.0f));
            float l2 = 0.0f;
#pragma unroll 1
            for (int c = 0; c < 8; c++) {
                uint32_t v[16], w[16];
                tmem_ld16(t_s + 16 * c, v);
                const float fk = f * page_ks[e][c], cw = page_vs[e][c] * cv;
                tmem_wait_ld();
                tmem_pin<16>(v);
#pragma unroll
                for (int k = 0; k < 16; k++) v[k] = __float_as_uint(ex2(fmaf(__uint_as_float(v[k]), fk, -mref)));
                if (!whole) {
                    const uint32_t mk = mask(c);
#pragma unroll
                    for (int k = 0; k < 16; k++) v[k] = (mk >> k) & 1u ? v[k] : 0u;
                }
#pragma unroll
                for (int k = 0; k < 16; k += 2) {
                    const float x = __uint_as_float(v[k]), y = __uint_as_float(v[k + 1]);
                    l += x;
                    l2 += y;
                    w[k / 2] = split_h2(x * cw, y * cw, w[8 + k / 2]);
                }
                // hi in columns 0-7 of the group's 16, lo in 8-15: only this group's scores are replaced
                tmem_st16(t_s + 16 * c, w);
            }
            l += l2;
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(pfull(grp));
            mbar_arrive(gempty(e));
            ok = mbar_wait(ofull(grp), (j >> 1) & 1, abortp, err, VXC_DERR_TIMEOUT_MMA);
            if (!__all_sync(0xffffffffu, ok)) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < HD / 32; c++) {
                uint32_t v[32];
                tmem_ld32(t_o + tl + 32 * c, v);
                tmem_wait_ld();
                tmem_pin<32>(v);
#pragma unroll
                for (int d = 0; d < 32; d++) acc[32 * c + d] += __uint_as_float(v[d]);
            }
            tc_fence_before();
            mbar_arrive(oempty(grp));
        }
        // join of the groups, outputs in units of 2^m.  Both groups have waited for their last
        // P V product, so no product reads shared memory any more (after an abort one may, but
        // then nothing is written).
        float *so = reinterpret_cast<float *>(sm + M::K);     // [HD][129]
        float *st = so + HD * 129;                            // [128][4]: group B's m and l, the result's M and L
        const float back = mv == -INFINITY ? 0.0f : ex2(fmaxf(fminf(mv - m - KV8_HEAD, 126.0f), -126.0f));
#pragma unroll
        for (int d = 0; d < HD; d++) acc[d] *= back;
        mn_group_sync();
        if (grp == 1) {
#pragma unroll
            for (int d = 0; d < HD; d++) so[d * 129 + row] = acc[d];
            st[4 * row] = m;
            st[4 * row + 1] = l;
        }
        mn_group_sync();
        if (grp == 0) {
            const float m1 = st[4 * row], l1 = st[4 * row + 1], mm = fmaxf(m, m1);
            const float e0 = m == -INFINITY ? 0.0f : ex2(m - mm), e1 = m1 == -INFINITY ? 0.0f : ex2(m1 - mm);
            const float L = e0 * l + e1 * l1;
            const float inv = ns > 1 ? 1.0f : L == 0.0f ? 0.0f : 1.0f / L;   // no token: 0; NaN stays
#pragma unroll
            for (int d = 0; d < HD; d++) so[d * 129 + row] = (e0 * acc[d] + e1 * so[d * 129 + row]) * inv;
            st[4 * row + 2] = mm;
            st[4 * row + 3] = L;
        }
        mn_group_sync();
        if (!*abortp) {
            // a warp per query, lanes over the head dim
            for (int i = warp - 4; i < 128 && q0 + i < nq; i += 8) {
                const int oq = q0 + i, orow = rq.row0 + oq / G, h = kvh * G + oq % G;
                float *rec = a.part + (((size_t)orow * a.H + h) * a.S + split) * (HD + 4);
                float *dst = ns > 1 ? rec + 4 : a.out + (size_t)orow * a.ldo + (size_t)h * HD;
#pragma unroll
                for (int d = lane; d < HD; d += 32) dst[d] = so[d * 129 + i];
                if (ns > 1 && lane == 0) *reinterpret_cast<float2 *>(rec) = make_float2(st[4 * i + 2], st[4 * i + 3]);
            }
        }
        asm volatile("setmaxnreg.dec.sync.aligned.u32 128;");
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        if (warp == 12 && lane == 0) {
            // ------------------------------ S = Q K^T ------------------------------
            const uint32_t idesc = (1u << 4) | ((uint32_t)(128 >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
#pragma unroll 1
            for (int j = 0; j < nt; j++) {
                const int s = j & 1;
                bool ok = mbar_wait(kfull(s), (j >> 1) & 1, abortp, err, VXC_DERR_TIMEOUT_TMA);
                // the buffer's weights (tile j - 2) have been multiplied
                if (ok && j >= 2) ok = mbar_wait(ofull(s), ((j >> 1) - 1) & 1, abortp, err, VXC_DERR_TIMEOUT_MMA);
                if (!ok) break;
                tc_fence_after();
                const uint32_t kb = smb + M::K + s * M::TILE, d = tmem + 128 * s;
#pragma unroll
                for (int k = 0; k < HD / 16; k++) {
                    const uint64_t bd = sdesc(kb + k * 2 * MN_CHUNK, MN_CHUNK, 128);
                    mma_f16_ts(d, t_q + 8 * k, bd, idesc, k != 0);
                    mma_f16_ts(d, t_q + 64 + 8 * k, bd, idesc, 1u);
                }
                mma_commit(kempty(s));
                mma_commit(sfull(s));
            }
        } else if (warp == 13 && lane == 0) {
            // ------------------------------ O = P V ------------------------------
            // V is MN-major (bit 16): 8-column chunks MN_CHUNK apart, groups of 8 tokens 128 bytes apart
            const uint32_t idesc = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
#pragma unroll 1
            for (int j = 0; j < nt; j++) {
                const int s = j & 1;
                bool ok = mbar_wait(vfull(s), (j >> 1) & 1, abortp, err, VXC_DERR_TIMEOUT_TMA);
                ok = ok && mbar_wait(pfull(s), (j >> 1) & 1, abortp, err, VXC_DERR_TIMEOUT_MMA);
                if (ok && j >= 1) ok = mbar_wait(oempty((j - 1) & 1), ((j - 1) >> 1) & 1, abortp, err, VXC_DERR_TIMEOUT_MMA);
                if (!ok) break;
                tc_fence_after();
                const uint32_t vb = smb + M::V + s * M::TILE, p = tmem + 128 * s;
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const uint64_t bd = sdesc(vb + k * 256, 128, MN_CHUNK);
                    mma_f16_ts(t_o, p + 16 * k, bd, idesc, k != 0);
                    mma_f16_ts(t_o, p + 16 * k + 8, bd, idesc, 1u);
                }
                mma_commit(vempty(s));
                mma_commit(ofull(s));
            }
        } else if (warp == 14 && lane < 8) {
            // ------------------------------ blocks and scales ------------------------------
            const int *trow = a.table + (size_t)r * a.max_blocks;
            for (int j = 0; j < nt; j++) {
                const int e = j % MN_PAGES;
                if (j >= MN_PAGES && !mbar_wait(gempty(e), ((j / MN_PAGES) - 1) & 1, abortp, err, VXC_DERR_TIMEOUT_EPI)) break;
                const int p = p0 + 128 * j + 16 * lane;
                long long at = -1;
                float ks = 0.0f, vs = 0.0f;
                if (p < rq.kvlen) {
                    const int blk = trow[p / bs];
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
                page_at[e][lane] = at;
                page_ks[e][lane] = ks;
                page_vs[e][lane] = vs;
                page_lv[e][lane] = lg2(vs);
                mbar_arrive(gfull(e));
            }
        }
        __syncwarp();
        asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
    }

    // ------------------------------ end ------------------------------
    if ((warp == 12 || warp == 13) && lane == 0 && *abortp) {
        // an aborted issuer's products may still run: wait for them (bounded)
        const uint32_t bar = bar0 + 8u * (warp == 12 ? 16 : 17);
        mma_commit(bar);
        const uint64_t t1 = vxc_globaltimer();
        while (!mbar_try(bar, 0) && vxc_globaltimer() - t1 < 100000000ull) {}
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 12) tmem_dealloc(tmem, 512u);
}

template <int TYPE>
static cudaError_t launch_many(const Kv8AttnArgs &a, int tiles, cudaStream_t st) {
    void (*f)(const Kv8AttnArgs) = nullptr;
    size_t smem = 0;
    switch (a.kv.head_dim) {
        case 32: f = k_kv8_attn_many<TYPE, 32>; smem = MnSmem<32>::BYTES; break;
        case 64: f = k_kv8_attn_many<TYPE, 64>; smem = MnSmem<64>::BYTES; break;
        case 96: f = k_kv8_attn_many<TYPE, 96>; smem = MnSmem<96>::BYTES; break;
        default: f = k_kv8_attn_many<TYPE, 128>; smem = MnSmem<128>::BYTES; break;
    }
    // TMEM is allocated whole: one CTA per SM, so at least half of the shared memory is asked for
    if (smem < 116 * 1024) smem = 116 * 1024;
    cudaError_t e = kv8_allow_smem((const void *)f, smem);
    if (e != cudaSuccess) return e;
    return kv8_launch(f, dim3(tiles, a.kv.n_kv_heads, a.S), dim3(MN_THREADS), smem, st, 1, a);
}

cudaError_t kv8_attn_many(const Kv8AttnArgs &a, int tiles, cudaStream_t st) {
    return a.kv.type == VXC_KV8_INT8 ? launch_many<VXC_KV8_INT8>(a, tiles, st) : launch_many<VXC_KV8_E4M3>(a, tiles, st);
}
