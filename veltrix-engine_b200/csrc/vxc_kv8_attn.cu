// vxc_kv8_attn.cu — causal attention over the paged 8-bit KV cache
// (reference src/model.c:299-338, over its fp32 cache).
//   out_i,h = sum_j softmax_j(scale q_i,h . k_j) v_j,  j <= position of row i
#include "vxc_kv8_attn.cuh"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

// ---------------------------------------------------------------------------
// Few queries per kv head (decode and small verify steps): split over the
// context, warp-level tensor instructions.
//
// CTA = (request, kv head) x one split of the request's tokens.  Queries are
// the request's rows times the heads of the kv head, query = row * G + head, so
// every byte of the split is read once for all.
// Each of the 4 warps goes over every fourth piece of 32 tokens (two tiles of
// 16), with a softmax state and an output of its own; the warps are joined at
// the end.
//
// Products.  mma m16n8k16 in fp16 with fp32 sums.  A code is exact in fp16.  A
// query row is scaled by a power of two and split into two fp16 parts, hi and
// lo (22 bits); so are the weights.
//   NQ = 8: rows 0-7 of the instruction's 16 are hi, rows 8-15 are lo, and
//     their two sums are added: one instruction does both products.
//   NQ = 16: two instructions into the same sums, hi and lo.
// Layouts.  The sum over the head dim may go in any order, so lane t of a quad
// takes the pieces of a K row that it can load as whole words (Kv8Few::k_at),
// and the query's fragment is loaded in the same order.  Likewise the output's
// columns: lane group g takes pieces of a V row (Kv8Few::v_at).  Scores come out
// where the weights' fragment wants them: lane (g, t) has tokens 2t, 2t+1,
// 2t+8, 2t+9 of query g, and reads V of just these.
// A tile (16 rows) is one contiguous span of its block; it comes by cp.async,
// 512 bytes an instruction, to the warp's own ring, its 16-byte chunks exchanged
// within 128 bytes so that both reads are free of bank conflicts at head dims 64
// and 128.  (With every lane fetching the bytes it uses itself an instruction
// touched 8 lines for K and 16 for V instead of 4, and issuing took a third of
// the time.)
// Softmax in base 2 with two running maxima per query: m of the scores s, for
// the sum l of 2^(s - m), and mv of s + log2(v_scale), the reference of the
// weights w = 2^(s - mv) v_scale 2^KV8_HEAD that multiply the codes of V: a
// weight keeps its 22 bits whatever the scales of the other blocks are.  They
// follow the true maximum only when it is over KV8_LAG ahead, so the output is
// seldom rescaled.
// Tokens behind the request's last one and blocks outside the cache are read
// as zeros (cp.async's zero fill), so nothing of theirs reaches a product.
// The blocks and scales of the split are looked up once, at the start.
//
// Measured (heads of 128): 33 requests of one row behind up to 16384 tokens, 64
// heads over 8, 102 us one call after the other, 5.3 TB/s of the cache's bytes
// (108 to 113 us among other work); 8 requests of 5 rows behind up to 768 tokens, 32
// heads, 13.9 us; 8 of one row, 32 heads of 64 over 4, 7.6 us.  Bound: bytes for
// long contexts (issue slots 40 %, tensor pipe 33 % busy).  Short ones: a CTA's
// latencies, about 4 us, and its warps' chain of scores, maxima, weights and
// products, 1.6 us per piece of 32 tokens with two warps per scheduler.
// ---------------------------------------------------------------------------
#define FEW_STAGES 2     // 32-token pieces per warp: one in use, one in flight (3: no faster, 4: fewer CTAs per SM, slower)

template <int HD>
struct Kv8Few {
    // pieces (bytes, count, place in the row) of a K row that lane t of a quad reads, of a V row that lane group g reads
    static constexpr int K = HD % 64 == 0 ? 16 : 8, NK = HD / 4 / K;
    static constexpr int V = HD == 128 ? 16 : HD == 64 ? 8 : 4, NV = HD / 8 / V;
    static __device__ __forceinline__ int k_at(int c, int t) { return c * 4 * K + t * K; }
    static __device__ __forceinline__ int v_at(int c, int g) { return c * 8 * V + g * V; }
    // place of byte `at` of row `row` in a tile of the ring (at a multiple of the piece)
    static __device__ __forceinline__ int k_slot(int row, int at) {
        const int b = row * HD + at;
        return HD == 128 ? b ^ ((row & 1) << 6) : b;
    }
    static __device__ __forceinline__ int v_slot(int row, int at) {
        const int b = row * HD + at;
        return HD == 128 ? b ^ ((row & 6) << 4) : HD == 64 ? b ^ ((row & 6) << 4) : b;
    }
};

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The splits of a request and head are joined by their cluster, through
// distributed shared memory, while a cluster holds them all (a.S <= 8); else
// they leave records in device memory for k_kv8_attn_join:
// [row][head][S][4 + HD] = {m, l, -, -, o[HD]}, l = sum of 2^(s - m), o = the split's own output.  (A split's
// output is divided by its own l and joined with weights 2^(m - M) l / L, a warp's by a power of two over l:
// sums of 2^(s - m) v themselves would overflow for V within their number of tokens of the largest float.)
template <int TYPE, int HD, int NQ>
__global__ void __launch_bounds__(128, 2) k_kv8_attn_few(const Kv8AttnArgs a) {
    using P = Kv8Few<HD>;
    constexpr int NR = NQ / 8;                 // query rows per lane
    constexpr int KS = HD / 16;                // steps over the head dim
    constexpr int NT = HD / 8;                 // column tiles of the output
    constexpr int TILE = HD * 32;              // bytes of K and V of 16 tokens
    constexpr int STAGE = 2 * TILE;
    extern __shared__ __align__(128) unsigned char sm[];
    const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int KH = a.kv.n_kv_heads, G = a.H / KH, bs = a.kv.block_size;
    pdl_trigger();
    pdl_wait();
    // (scratch in the ring: static shared memory would move the ring off its 128-byte lines, +6 %)
    const int kvh = blockIdx.y, split = blockIdx.x, place = (int)blockIdx.z / a.chunks;
    const int q0 = ((int)blockIdx.z - place * a.chunks) * NQ;   // first query of the CTA
    const int r = a.ranked ? kv8_ranked(a, place, reinterpret_cast<int *>(sm)) : place;
    const Kv8Req rq = kv8_req(a, r);
    if (rq.over && kvh == 0 && split == 0 && q0 == 0 && tid == 0) vxc_flag_error(a.err, VXC_DERR_BAD_BLOCK);
    const int nq = min(rq.T * G - q0, NQ);
    if (nq <= 0) return;
    int SL;
    const int ns = kv8_splits(rq.kvlen, a.sl_min, a.S, SL);
    if (split >= ns) return;
    const int p0 = split * SL, p1 = min(p0 + SL, rq.pos + (q0 + nq - 1) / G + 1);

    // blocks (-1: outside the cache) of the split, then their {K scale, V scale, its logarithm}
    const int e0 = p0 / bs, ne = p1 > p0 ? (p1 - 1) / bs - e0 + 1 : 0;
    int *page_id = reinterpret_cast<int *>(sm + 4 * FEW_STAGES * STAGE);
    float4 *page = reinterpret_cast<float4 *>(page_id + a.pages);
    const int *trow = rq.table + e0;
    for (int i = tid; i < ne; i += 128) {
        int b = trow[i];
        if (b < 0 || b >= a.kv.n_blocks) {
            b = -1;
            vxc_flag_error(a.err, VXC_DERR_BAD_BLOCK);
        }
        page_id[i] = b;
    }

    // pieces w, w + 4, ... of 32 tokens: 2 tiles each
    const int npc = p1 > p0 ? (p1 - p0 + 31) >> 5 : 0, nit = npc > w ? (npc - w + 3) >> 2 : 0;
    unsigned char *ring = sm + w * (FEW_STAGES * STAGE);
    const uint32_t ring_u = smem_u32(ring);
    const int bs16 = bs >> 4;
    const uint8_t *kb = (const uint8_t *)a.kv.k + (size_t)kvh * bs * HD + lane * 16;
    const uint8_t *vb = (const uint8_t *)a.kv.v + (size_t)kvh * bs * HD + lane * 16;
    const size_t bstep = (size_t)KH * bs * HD;
    const int tile0 = p0 / 16 - e0 * bs16 + 2 * w;   // the warp's first tile, counted from the first page's start
    int pi = tile0 / bs16, oi = tile0 % bs16;        // page and tile in it of the next tile to bring in
    int pc = pi, oc = oi;                            // and of the next one to use
    int p_in = p0 + 32 * w;
    __syncthreads();   // page_id
    auto issue = [&](int it) {
        if (it < nit) {
            uint32_t dst = ring_u + it % FEW_STAGES * STAGE;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int blk = p_in < p1 ? page_id[pi] : -1;
                const size_t at = (size_t)max(blk, 0) * bstep + (size_t)(oi * 16) * HD;
                const uint8_t *ks = kb + at, *vs = vb + at;
                const int live = blk >= 0 ? rq.kvlen - p_in : 0;   // tokens of the tile that exist
                // instruction k brings chunks 32 k + lane of the span
                auto bring = [&](auto copy) {
#pragma unroll
                    for (int k = 0; k < HD / 32; k++) {
                        const int byte = k * 512 + lane * 16, row = byte / HD, in = byte % HD;
                        copy(dst + P::k_slot(row, in), ks + k * 512, row);
                        copy(dst + HD * 16 + P::v_slot(row, in), vs + k * 512, row);
                    }
                };
                if (live >= 16) bring([](uint32_t d, const uint8_t *x, int) { cp_async<16>(d, x); });
                else bring([&](uint32_t d, const uint8_t *x, int row) { cp_async_zfill<16>(d, x, row < live); });
                dst += TILE;
                p_in += 16;
                oi += u == 0 ? 1 : 7;   // the pair's second tile; the warp's next piece
                while (oi >= bs16) oi -= bs16, pi++;
            }
            p_in += 96;
        }
        cp_commit();
    };
    if (nit > 0) {
#pragma unroll 1
        for (int i = 0; i < FEW_STAGES - 1; i++) issue(i);
    }
    for (int i = tid; i < ne; i += 128) {
        const int b = page_id[i];
        float4 e = make_float4(0.0f, 0.0f, -INFINITY, 0.0f);
        if (b >= 0) {
            const size_t bh = (size_t)b * KH + kvh;
            e.x = a.kv.k_scale[bh];
            e.y = a.kv.v_scale[bh];
            e.z = lg2(e.y);
        }
        page[i] = e;
    }

    // queries: fragments hi (and lo), the factor of each row's scores
    uint32_t qf[NR == 1 ? 1 : 2][KS][4];
    float f[NR];
    int lim[NR];   // last visible token
#pragma unroll
    for (int i = 0; i < NR; i++) {
        const int q = g + 8 * i;
        const bool have = q < nq;
        const int row = rq.row0 + (have ? (q0 + q) / G : 0), h = kvh * G + (have ? (q0 + q) % G : 0);
        const float *x = a.q + (size_t)row * a.ldq + (size_t)h * HD;
        float4 v[KS];
        float mx = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const int c = s / (P::K / 4), e = P::k_at(c, t) + 4 * (s % (P::K / 4));
            v[s] = have ? *reinterpret_cast<const float4 *>(x + e) : make_float4(0.f, 0.f, 0.f, 0.f);
            mx = fmaxf(mx, fmaxf(fmaxf(fabsf(v[s].x), fabsf(v[s].y)), fmaxf(fabsf(v[s].z), fabsf(v[s].w))));
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        // the row's largest element into [2^13, 2^14)
        const int ex = min(max((int)(__float_as_uint(mx) >> 23), 14), 253);
        const float up = __uint_as_float((uint32_t)(267 - ex) << 23), down = __uint_as_float((uint32_t)(ex - 13) << 23);
        f[i] = a.scale * 1.4426950408889634f * down;
        lim[i] = have ? rq.pos + (q0 + q) / G : -1;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            uint32_t l0, l1;
            const uint32_t h0 = split_h2(v[s].x * up, v[s].y * up, l0), h1 = split_h2(v[s].z * up, v[s].w * up, l1);
            if (NR == 1) {
                qf[0][s][0] = h0, qf[0][s][1] = l0, qf[0][s][2] = h1, qf[0][s][3] = l1;
            } else {
                qf[0][s][i] = h0, qf[0][s][2 + i] = h1;
                qf[NR - 1][s][i] = l0, qf[NR - 1][s][2 + i] = l1;
            }
        }
    }

    float o[NT][4];
#pragma unroll
    for (int j = 0; j < NT; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
    float m[NR], mv[NR], l[NR];
#pragma unroll
    for (int i = 0; i < NR; i++) m[i] = mv[i] = -INFINITY, l[i] = 0.0f;

    __syncthreads();   // page
#pragma unroll 1
    for (int it = 0; it < nit; it++) {
        __syncwarp();   // every lane has read the piece that is replaced
        issue(it + FEW_STAGES - 1);
        cp_wait<FEW_STAGES - 1>();
        __syncwarp();   // every lane's copies have landed
        const unsigned char *stg = ring + (it % FEW_STAGES) * STAGE;
        const int p = p0 + 32 * (w + 4 * it) + 2 * t;   // lane's tokens p, p + 1, p + 8, p + 9 of each tile
        // scores
        float sc[2][2][4], ksc[2], vsc[2], lv[2];
        bool none[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const bool in = p0 + 32 * (w + 4 * it) + 16 * u < p1;
            const float4 e = in ? page[pc] : make_float4(0.0f, 0.0f, -INFINITY, 0.0f);
            none[u] = !in || page_id[pc] < 0;
            ksc[u] = e.x, vsc[u] = e.y, lv[u] = e.z;
            oc += u == 0 ? 1 : 7;
            while (oc >= bs16) oc -= bs16, pc++;
#pragma unroll
            for (int n = 0; n < 2; n++) sc[u][n][0] = sc[u][n][1] = sc[u][n][2] = sc[u][n][3] = 0.0f;
        }
#pragma unroll
        for (int u = 0; u < 2; u++) {
#pragma unroll
            for (int c = 0; c < P::NK; c++) {
                uint32_t word[2][P::K / 4];
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    const unsigned char *src = stg + u * TILE + n * 8 * HD + P::k_slot(g, P::k_at(c, t));
                    if (P::K == 16) {
                        const uint4 x = *reinterpret_cast<const uint4 *>(src);
                        word[n][0] = x.x, word[n][1] = x.y, word[n][P::K / 4 - 2] = x.z, word[n][P::K / 4 - 1] = x.w;
                    } else {
                        const uint2 x = *reinterpret_cast<const uint2 *>(src);
                        word[n][0] = x.x, word[n][1] = x.y;
                    }
                }
#pragma unroll
                for (int e = 0; e < P::K / 4; e++) {
                    const int s = c * (P::K / 4) + e;
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        uint32_t b0, b1;
                        codes_h2<TYPE>(word[n][e], b0, b1);
                        mma16816(sc[u][n], qf[0][s], b0, b1);
                        if (NR == 2) mma16816(sc[u][n], qf[NR - 1][s], b0, b1);
                    }
                }
            }
        }
        // weights
        uint32_t wf[2][NR == 1 ? 1 : 2][4];
#pragma unroll
        for (int i = 0; i < NR; i++) {
            float s[2][4], mx[2];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const float fk = f[i] * ksc[u];
                const float (&x)[2][4] = sc[u];
                if (NR == 1) {
                    s[u][0] = x[0][0] + x[0][2], s[u][1] = x[0][1] + x[0][3];
                    s[u][2] = x[1][0] + x[1][2], s[u][3] = x[1][1] + x[1][3];
                } else {
                    s[u][0] = x[0][2 * i], s[u][1] = x[0][2 * i + 1], s[u][2] = x[1][2 * i], s[u][3] = x[1][2 * i + 1];
                }
                const int end = none[u] ? -1 : lim[i];
#pragma unroll
                for (int k = 0; k < 4; k++)
                    s[u][k] = p + 16 * u + (k & 1) + (k >> 1) * 8 <= end ? s[u][k] * fk : -INFINITY;
                mx[u] = fmaxf(fmaxf(s[u][0], s[u][1]), fmaxf(s[u][2], s[u][3]));
            }
            float mm = fmaxf(mx[0], mx[1]), mxv = fmaxf(mx[0] + lv[0], mx[1] + lv[1]);
            mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, 1));
            mxv = fmaxf(mxv, __shfl_xor_sync(0xffffffffu, mxv, 1));
            mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, 2));
            mxv = fmaxf(mxv, __shfl_xor_sync(0xffffffffu, mxv, 2));
            if (mm > m[i] + KV8_LAG || (m[i] == -INFINITY && mm > m[i])) {
                l[i] *= ex2(m[i] - mm);   // 0 at first
                m[i] = mm;
            }
            float shrink = 1.0f;
            const float least = m[i] - KV8_FLOOR;
            mxv = fmaxf(mxv, least);
            if (mxv > mv[i] + KV8_LAG || least > mv[i]) {
                shrink = ex2(mv[i] - mxv);
                mv[i] = mxv;
            }
            if (__any_sync(0xffffffffu, shrink != 1.0f)) {
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    if (NR == 1) {
                        o[j][0] *= shrink, o[j][1] *= shrink, o[j][2] *= shrink, o[j][3] *= shrink;
                    } else {
                        o[j][2 * i] *= shrink, o[j][2 * i + 1] *= shrink;
                    }
                }
            }
            float mref = m[i] == -INFINITY ? 0.0f : m[i];
            float cv = ex2(fminf(mref - mv[i] + KV8_HEAD, KV8_FLOOR + KV8_HEAD));   // (no token yet: mv is -inf)
            const float unit = kv8_unit(fmaxf(vsc[0], vsc[1]), cv, mref);
            float sum = 0.0f;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const float c = kv8_factor(vsc[u], cv);
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    s[u][k] = ex2(s[u][k] - mref);
                    sum += s[u][k];
                    s[u][k] *= c;
                }
                uint32_t l0, l1;
                const uint32_t h0 = split_h2(s[u][0], s[u][1], l0), h1 = split_h2(s[u][2], s[u][3], l1);
                if (NR == 1) {
                    wf[u][0][0] = h0, wf[u][0][1] = l0, wf[u][0][2] = h1, wf[u][0][3] = l1;
                } else {
                    wf[u][0][i] = h0, wf[u][0][2 + i] = h1;
                    wf[u][NR - 1][i] = l0, wf[u][NR - 1][2 + i] = l1;
                }
            }
            l[i] = fmaf(sum, unit, l[i]);
        }
        // weights times V: byte j of the lane's piece of tokens 2t, 2t+1, 2t+8, 2t+9 is column tile j
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const unsigned char *vst = stg + u * TILE + HD * 16;
#pragma unroll
            for (int c = 0; c < P::NV; c++) {
                uint32_t tok[4][P::V / 4];
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    const unsigned char *src = vst + (n >> 1) * 8 * HD + P::v_slot(2 * t + (n & 1), P::v_at(c, g));
                    if (P::V == 16) {
                        const uint4 x = *reinterpret_cast<const uint4 *>(src);
                        tok[n][0] = x.x, tok[n][P::V / 4 > 1 ? 1 : 0] = x.y;
                        tok[n][P::V / 4 > 2 ? 2 : 0] = x.z, tok[n][P::V / 4 - 1] = x.w;
                    } else if (P::V == 8) {
                        const uint2 x = *reinterpret_cast<const uint2 *>(src);
                        tok[n][0] = x.x, tok[n][P::V / 4 - 1] = x.y;
                    } else {
                        tok[n][0] = *reinterpret_cast<const uint32_t *>(src);
                    }
                }
#pragma unroll
                for (int e = 0; e < P::V / 4; e++) {
                    uint32_t b0[4], b1[4];
                    codes_h2<TYPE>(__byte_perm(tok[0][e], tok[1][e], 0x5140), b0[0], b0[1]);
                    codes_h2<TYPE>(__byte_perm(tok[0][e], tok[1][e], 0x7362), b0[2], b0[3]);
                    codes_h2<TYPE>(__byte_perm(tok[2][e], tok[3][e], 0x5140), b1[0], b1[1]);
                    codes_h2<TYPE>(__byte_perm(tok[2][e], tok[3][e], 0x7362), b1[2], b1[3]);
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int j = c * P::V + 4 * e + k;
                        mma16816(o[j], wf[u][0], b0[k], b1[k]);
                        if (NR == 2) mma16816(o[j], wf[u][NR - 1], b0[k], b1[k]);
                    }
                }
            }
        }
    }
    cp_wait<0>();
    __syncthreads();   // the ring is free

    // join the warps: their outputs, maxima and sums
    float *so = reinterpret_cast<float *>(sm);            // [4][NQ][HD + 4]
    float *sml = so + 4 * NQ * (HD + 4);                  // [4][NQ][2]
#pragma unroll
    for (int i = 0; i < NR; i++) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        const float back = mv[i] == -INFINITY ? 0.0f : ex2(mv[i] - m[i] - KV8_HEAD);
        const float inv = kv8_pow2_under(l[i]);
        float *dst = so + (w * NQ + g + 8 * i) * (HD + 4);
#pragma unroll
        for (int j = 0; j < NT; j++) {
            const int c = j / P::V, e = j % P::V;
            const float x = NR == 1 ? o[j][0] + o[j][2] : o[j][2 * i], y = NR == 1 ? o[j][1] + o[j][3] : o[j][2 * i + 1];
            dst[P::v_at(c, 2 * t) + e] = x * inv * back;
            dst[P::v_at(c, 2 * t + 1) + e] = y * inv * back;
        }
        if (t == 0) {
            sml[(w * NQ + g + 8 * i) * 2] = m[i];
            sml[(w * NQ + g + 8 * i) * 2 + 1] = l[i];
        }
    }
    __syncthreads();
    // the CTA's result, one warp per query: {m, l, -, -, o[HD]}
    const bool cluster = a.S <= 8;
    float *res = sml + 4 * NQ * 2;                        // [NQ][HD + 4]
    for (int q = w; q < nq; q += 4) {
        float M = -INFINITY, mw[4], L = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; k++) M = fmaxf(M, mw[k] = sml[(k * NQ + q) * 2]);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float l = sml[(k * NQ + q) * 2 + 1];
            mw[k] = mw[k] == -INFINITY ? 0.0f : ex2(mw[k] - M);
            L += mw[k] * l;
            mw[k] *= kv8_pow2_over(l);
        }
        const int row = rq.row0 + (q0 + q) / G, h = kvh * G + (q0 + q) % G;
        float *rec = cluster ? res + q * (HD + 4) : a.part + (((size_t)row * a.H + h) * a.S + split) * (HD + 4);
        float *out = a.out + (size_t)row * a.ldo + (size_t)h * HD;
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;   // no token: 0; NaN stays
#pragma unroll
        for (int k = 0; k < 4; k++) mw[k] *= inv;
#pragma unroll
        for (int d = lane; d < HD; d += 32) {
            float x = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (mw[k] != 0.0f) x = fmaf(mw[k], so[(k * NQ + q) * (HD + 4) + d], x);
            if (ns == 1) out[d] = x;
            else rec[4 + d] = x;
        }
        if (ns > 1 && lane == 0) *reinterpret_cast<float2 *>(rec) = make_float2(M, L);
    }
    if (!cluster || ns == 1) return;
    // every CTA of the cluster that got here has ns splits: they share out the queries
    cg::cluster_group cl = cg::this_cluster();
    cl.sync();
    for (int q = split + ns * w; q < nq; q += 4 * ns) {
        float M = -INFINITY, L = 0.0f, x[HD / 32];
        float2 ml[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            if (k < ns) {
                ml[k] = *reinterpret_cast<const float2 *>(cl.map_shared_rank(res + q * (HD + 4), k));
                M = fmaxf(M, ml[k].x);
            }
        }
#pragma unroll
        for (int k = 0; k < 8; k++) {
            if (k < ns) {
                ml[k].y *= ml[k].x == -INFINITY ? 0.0f : ex2(ml[k].x - M);
                L += ml[k].y;
            }
        }
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
        for (int d = 0; d < HD / 32; d++) x[d] = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            if (k < ns) {
                const float *rec = cl.map_shared_rank(res + q * (HD + 4), k);
                const float e = ml[k].y * inv;
#pragma unroll
                for (int d = 0; d < HD / 32; d++) x[d] = fmaf(e, rec[4 + d * 32 + lane], x[d]);
            }
        }
        float *out = a.out + (size_t)(rq.row0 + q / G) * a.ldo + (size_t)(kvh * G + q % G) * HD;
#pragma unroll
        for (int d = 0; d < HD / 32; d++) out[d * 32 + lane] = x[d];
    }
    cl.sync();   // the others have read this CTA's results
}

// Joins the splits of the requests that have several: one warp per (row, head).
template <int HD>
__global__ void __launch_bounds__(128) k_kv8_attn_join(const Kv8AttnArgs a) {
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_trigger();
    pdl_wait();
    const int i = blockIdx.x, h = blockIdx.y * 4 + w;
    if (h >= a.H || i >= kv8_row0(a, a.n_req)) return;
    int lo = 0, hi = a.n_req;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (kv8_row0(a, mid) <= i) lo = mid; else hi = mid;
    }
    const Kv8Req rq = kv8_req(a, lo);
    if (i - rq.row0 < 0 || i - rq.row0 >= rq.T) return;
    int SL;
    const int ns = kv8_splits(rq.kvlen, a.sl_min, a.S, SL);
    if (ns == 1) return;
    // only the splits that begin at or before the row's own token hold anything
    const int live = min(ns, (rq.pos + (i - rq.row0)) / SL + 1);
    const float *rec = a.part + ((size_t)i * a.H + h) * a.S * (HD + 4);
    const int n = rq.pos + (i - rq.row0) >= 0 ? live : 0;
    float M = -INFINITY, L = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto head = [&](int s) { return *reinterpret_cast<const float2 *>(rec + (size_t)s * (HD + 4)); };
    auto unit = [&](float m) { return m == -INFINITY ? 0.0f : ex2(m - M); };   // 2^m in units of 2^M
    for (int s = lane; s < n; s += 32) M = fmaxf(M, head(s).x);
#pragma unroll
    for (int k = 16; k; k >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, k));
    for (int s = lane; s < n; s += 32) L = fmaf(unit(head(s).x), head(s).y, L);
#pragma unroll
    for (int k = 16; k; k >>= 1) L += __shfl_xor_sync(0xffffffffu, L, k);
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;   // no token: 0; NaN stays
    // lanes have a record's {m, l} each, then, of one record after the other, four values each
    const float *mine = rec + 4 + 4 * min(lane, HD / 4 - 1);
    for (int at = 0; at < n; at += 32) {
        const int some = min(n - at, 32);
        const float2 ml = lane < some ? head(at + lane) : make_float2(-INFINITY, 0.0f);
        const float w = unit(ml.x) * ml.y * inv;
#pragma unroll 8
        for (int s = 0; s < some; s++) {
            const float e = __shfl_sync(0xffffffffu, w, s);
            const float4 x = *reinterpret_cast<const float4 *>(mine + (size_t)(at + s) * (HD + 4));
            if (e != 0.0f) o.x = fmaf(e, x.x, o.x), o.y = fmaf(e, x.y, o.y), o.z = fmaf(e, x.z, o.z), o.w = fmaf(e, x.w, o.w);
        }
    }
    if (lane < HD / 4) *reinterpret_cast<float4 *>(a.out + (size_t)i * a.ldo + (size_t)h * HD + 4 * lane) = o;
}

static int attn_check(const vxc_kv8 *kv, int n_heads, int n_req, int n_rows, int max_new, int max_blocks) {
    if (int rc = vxc_kv8_check(kv, "vxc_kv8_attn")) return rc;
    if (n_heads < 1 || n_heads > 65535 || n_heads % kv->n_kv_heads) {
        vxc_set_error("vxc_kv8_attn: %d heads over %d kv heads", n_heads, kv->n_kv_heads);
        return -4;
    }
    if (n_req < 1 || n_req > VXC_KV8_MAX_REQ || n_rows < 0 || n_rows > VXC_KV8_MAX_ROWS || max_new < 1 ||
        max_blocks < 1 || (long long)max_blocks * kv->block_size > KV8_MAX_TOKENS ||
        (long long)n_rows * n_heads > INT_MAX) {
        vxc_set_error("vxc_kv8_attn: %d requests, %d rows (%d of one request), %d blocks per request", n_req, n_rows,
                      max_new, max_blocks);
        return -4;
    }
    return 0;
}

// How a call is cut: kernel, queries per CTA and splits.
struct AttnPlan {
    int nq;        // queries per CTA: 8 or 16 (k_kv8_attn_few), 32, 64 or 128 (k_kv8_attn_many)
    int chunks;    // k_kv8_attn_few: CTAs for a request's queries
    int tiles;     // k_kv8_attn_many: tiles of all requests at most
    int S, sl_min;
    int pages;     // blocks a split may touch (k_kv8_attn_few)
};
#ifndef ATTN_FEW_MAX
#define ATTN_FEW_MAX 16   // queries of a request and kv head up to which k_kv8_attn_few is used
#endif

// The host knows the width of the table, not the lengths behind it: they are taken as spread evenly from
// nothing to that width.  Where they are not (us; table as wide as the longest request, of 4096, of 16384
// tokens): 8 requests of 5 rows behind 763 tokens, 32 heads, 14.7, 23, 23; 8 of one row, 32 heads of 64 over 4,
// 7.5, 7.7, 7.7; 8 of 17 rows 36, 37, 37; 32 of 7 rows, all behind 4089 tokens, 64 heads over 8, 133 or, with
// one block more, 145, 146; 100 of 26 rows in 26 tokens, 28 heads of 32, 62, 59, 131.
#define ATTN_FILL 0.5

static AttnPlan attn_plan(const vxc_kv8 *kv, int n_heads, int n_req, int n_rows, int max_new, int max_blocks) {
    AttnPlan p;
    p.chunks = 1;
    const int G = n_heads / kv->n_kv_heads;
    const long long most = (long long)(max_new < n_rows ? max_new : n_rows) * G;   // queries of a request
    const long long tokens = (long long)max_blocks * kv->block_size;
    long long units, S;
    if (most <= ATTN_FEW_MAX) {
        p.nq = most <= 8 ? 8 : 16;
        p.tiles = 0;
        units = (long long)n_req * kv->n_kv_heads;
        // A CTA costs about 4 us besides its tokens and, joined by a cluster, 2 us more; two fit an SM, a
        // cluster's on one of 8 groups of 16 SMs or more, and each further CTA of a unit takes 12 us of a place
        // (a cluster's CTAs begin and end together); above 8 a second kernel joins them.  The S of the least
        // time, as below; measured (us, S = 1, 2, ...): 256 units of 768 tokens 13.5, 17.5; 256 of 4096 58, 47,
        // 53; 512 of 8192 108, 127, 157; 800 of 4096 105, 136, 146; 264 of 16384 -, 105, 120, 138; 32 of 768
        // 9.2, in six 7.3; 48 of 2000 in five 12.8, in six 18.5 (not all of those clusters fit at once).
        p.sl_min = 128;
        double best = 0;
        const double byte = kv->head_dim / 128.0;
        S = 1;
        for (int i = 1; i <= 64; i++) {
            const double cta = 4 + 0.0125 * byte * tokens / i + (i == 1 ? 0 : i <= 8 ? 2 : 8);
            const double places = i <= 8 ? 4 + 12.0 * (i - 1) : 6.0 * i;
            const long long room = i == 1 || i > 8 ? 296 / i : 8 * (32 / i);   // units that fit at once
            const double all = n_req == 1 ? (units + room - 1) / room * cta
                                          : units * (places + ATTN_FILL * 0.0144 * byte * tokens) / 296 + 0.25 * cta;
            const double time = cta > all || units <= room ? cta : all;
            if (i == 1 || time < best) best = time, S = i;
        }
    } else {
        p.nq = most <= 32 ? 32 : most <= 64 ? 64 : 128;
        const long long full = (long long)n_rows * G / p.nq;
        // (a request per tile where all fit one; else tiles begin where k_kv8_attn_many says)
        p.tiles = (int)(most <= p.nq ? n_req : full + n_req);
        p.sl_min = 256;
        const long long busy = n_req < n_rows ? n_req : n_rows;
        const long long some = ((long long)n_rows * G + p.nq - 1) / p.nq;
        units = (some > busy ? some : busy) * kv->n_kv_heads;
        // A CTA costs about 11 us and 1.86 us per 128 tokens (at head dim 128; smaller heads and tiles, whose
        // tiles cost little less, are not told apart), one fits an SM; the join 3 us and its
        // records' way.  The S of the least time, as long as the longest CTA and as all of them on
        // 148 SMs: requests begin longest first and have ATTN_FILL of the tokens on average; a single one has
        // them all, and then CTAs come in whole rounds.  Measured (us, S = 1, 2, ...): 96 units of 8192
        // tokens 129, 78, 83; 64 units 128, 76, 59, 58, 62; 256 units of 4096 89, 112, 123; 200 units of
        // 16384 255, 212, 219; 128 units of 2000 39, 44, 54.
        double best = 0;
        S = 1;
        for (int i = 1; i <= 64; i++) {
            const double cta = 11 + 0.0145 * tokens / i;
            const double all = n_req == 1 ? (units * i + 147) / 148 * cta : units * (11.0 * i + ATTN_FILL * 0.0145 * tokens) / 148;
            const double join = i == 1 ? 0 : 3 + 2e-6 * n_rows * n_heads * i * (kv->head_dim + 4);
            const double time = (cta > all ? cta : all) + join;
            if (i == 1 || time < best) best = time, S = i;
        }
        // Many requests of few tokens: k_kv8_attn_few's CTAs, of 16 queries each, cost less (6.5 us besides
        // their tokens in a queue of them; 2 fit an SM, 3 with heads of 64, 4 with heads of 32).  100 requests
        // of 26 rows in 26 tokens, 28 heads of 32: 389 us in tiles, 46 so.  Where the estimates are near each
        // other the tile is kept: 43 requests of 16 rows in 51 tokens, 30 heads of 128 over 10, 32 and 33 us.
        const long long chunks = (most + 15) / 16;
        const double byte = kv->head_dim / 128.0, cta = 4 + 0.0125 * byte * tokens;
        const int places = 148 * (kv->head_dim >= 96 ? 2 : kv->head_dim == 64 ? 3 : 4);
        const double all = (double)n_req * kv->n_kv_heads * chunks * (6.5 + ATTN_FILL * 0.0144 * byte * tokens) / places + 0.25 * cta;
        if (tokens <= 8192 && chunks * n_req <= 65535 && (cta > all ? cta : all) < 0.8 * best) {
            p.nq = 16;
            p.chunks = (int)chunks;
            p.sl_min = (int)((tokens + 127) & ~127ll);
            S = 1;
        }
    }
    const long long need = (tokens + p.sl_min - 1) / p.sl_min;
    if (S > need) S = need;
    // k_kv8_attn_few: a tensor core's sums lose up to an ulp per step: 8192 tokens are 128 steps per
    // warp, 5e-6 at most
    const long long least = p.nq <= ATTN_FEW_MAX ? (tokens + 8191) / 8192 : 1;
    if (S > 64) S = 64;
    if (S < least) S = least;
    p.S = (int)(S < 1 ? 1 : S);
    // tokens of a split at most (kv8_splits)
    const long long even = (tokens + p.S - 1) / p.S, sl_max = ((even > p.sl_min ? even : p.sl_min) + 127) & ~127ll;
    p.pages = (int)(sl_max / kv->block_size + 2 + 3) & ~3;
    return p;
}

// Whether the splits leave records for k_kv8_attn_join.
static bool attn_records(const AttnPlan &p) { return p.S > (p.nq > ATTN_FEW_MAX ? 1 : 8); }

static size_t attn_need(const vxc_kv8 *kv, int n_heads, int n_rows, const AttnPlan &p) {
    return attn_records(p) ? (size_t)n_rows * n_heads * p.S * (kv->head_dim + 4) * sizeof(float) : 0;
}

extern "C" size_t vxc_kv8_attn_workspace_bytes(const vxc_kv8 *kv, int n_heads, int n_req, int n_rows, int max_new,
                                               int max_blocks) {
    if (attn_check(kv, n_heads, n_req, n_rows, max_new, max_blocks)) return 0;
    return attn_need(kv, n_heads, n_rows, attn_plan(kv, n_heads, n_req, n_rows, max_new, max_blocks));
}

typedef void (*attn_kernel_t)(const Kv8AttnArgs);
template <int TYPE, int HD>
static attn_kernel_t few_kernel(int nq) { return nq == 8 ? k_kv8_attn_few<TYPE, HD, 8> : k_kv8_attn_few<TYPE, HD, 16>; }
template <int TYPE>
static attn_kernel_t few_kernel(int hd, int nq) {
    switch (hd) {
        case 32: return few_kernel<TYPE, 32>(nq);
        case 64: return few_kernel<TYPE, 64>(nq);
        case 96: return few_kernel<TYPE, 96>(nq);
        default: return few_kernel<TYPE, 128>(nq);
    }
}
static attn_kernel_t join_kernel(int hd) {
    switch (hd) {
        case 32: return k_kv8_attn_join<32>;
        case 64: return k_kv8_attn_join<64>;
        case 96: return k_kv8_attn_join<96>;
        default: return k_kv8_attn_join<128>;
    }
}

// The launches of a call whose arguments hold.
static int attn_run(const Kv8AttnArgs &args, const AttnPlan &p, cudaStream_t st) {
    Kv8AttnArgs a = args;
    a.S = p.S;
    a.sl_min = p.sl_min;
    a.chunks = p.chunks;
    a.pages = p.pages;
    // the order is of no use where all CTAs fit the GPU at once, one or two per SM; its cost, a load and
    // n_req comparisons per CTA, is more than it gives where there are many more or contexts are short
    const bool many = p.nq > ATTN_FEW_MAX;
    const long long ctas = (long long)a.n_req * a.kv.n_kv_heads * p.S * p.chunks, at_once = many ? 148 : 2 * 148;
    a.ranked = (!many || p.tiles == a.n_req) && a.n_req > 1 && a.n_req <= KV8_RANKED && ctas > at_once && ctas <= 4 * at_once &&
               (long long)a.max_blocks * a.kv.block_size > 512;
    a.err = vxc_device_error_ptr();
    const vxc_kv8 *kv = &a.kv;
    const int hd = kv->head_dim;
    if (many) {
        VXC_CUDA_OK(kv8_attn_many(a, p.nq, p.tiles, st));
    } else {
        attn_kernel_t f = kv->type == VXC_KV8_INT8 ? few_kernel<VXC_KV8_INT8>(hd, p.nq) : few_kernel<VXC_KV8_E4M3>(hd, p.nq);
        size_t smem = (size_t)4 * FEW_STAGES * (hd * 64) + (size_t)p.pages * (sizeof(int) + sizeof(float4));
        const size_t join = ((size_t)4 * p.nq * (hd + 6) + (size_t)p.nq * (hd + 4)) * sizeof(float);
        if (smem < join) smem = join;
        VXC_CUDA_OK(kv8_allow_smem((const void *)f, smem));
        VXC_CUDA_OK(kv8_launch(f, dim3(p.S, kv->n_kv_heads, a.n_req * p.chunks), dim3(128), smem, st,
                               p.S <= 8 ? p.S : 1, a));
    }
    if (attn_records(p))
        VXC_CUDA_OK(kv8_launch(join_kernel(hd), dim3(a.n_rows, (a.H + 3) / 4), dim3(128), 0, st, 1, a));
    return 0;
}

extern "C" int vxc_kv8_attn(const vxc_kv8 *kv, const float *q, long long ldq, int n_heads, float scale,
                            const int *d_table, int max_blocks, const int *d_row0, const int *d_pos, int n_req,
                            int n_rows, int max_new, float *out, long long ldo, void *workspace,
                            size_t workspace_bytes, void *stream) {
    if (int rc = attn_check(kv, n_heads, n_req, n_rows, max_new, max_blocks)) return rc;
    const long long width = (long long)n_heads * kv->head_dim;
    if (!d_table || !d_row0 || !d_pos || !kv8_words(d_table, d_row0, d_pos) ||
        (n_rows > 0 && (!q || !out || (uintptr_t)q % 16 || (uintptr_t)out % 16 || ldq < width || ldo < width ||
                        ldq % 4 || ldo % 4))) {
        vxc_set_error("vxc_kv8_attn: an array is missing or not aligned, or rows are shorter than %lld floats", width);
        return -4;
    }
    if (!(scale == scale) || scale - scale != 0.0f) {
        vxc_set_error("vxc_kv8_attn: scale is not finite");
        return -4;
    }
    const AttnPlan p = attn_plan(kv, n_heads, n_req, n_rows, max_new, max_blocks);
    const size_t need = attn_need(kv, n_heads, n_rows, p);
    if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)) {
        vxc_set_error("vxc_kv8_attn: workspace of %zu bytes needed (16-byte aligned)", need);
        return -4;
    }
    if (int rc = vxc_require_device()) return rc;
    if (n_rows == 0) return 0;
    const Kv8AttnArgs a = {*kv, q, ldq, n_heads, scale, d_table, max_blocks, d_row0, d_pos, NULL, n_req, n_rows, max_new,
                           out, ldo, (float *)workspace};
    return attn_run(a, p, (cudaStream_t)stream);
}

// The forward's form: n_groups groups of rows_per_group rows, group g at
// position d_pos[g] with the blocks of table row d_seq[g] (none if negative).
int vxc_kv8_attn_groups(const vxc_kv8 *kv, const float *q, int n_heads, float scale, const int *d_table, int max_blocks,
                        const int *d_seq, const int *d_pos, int n_groups, int rows_per_group, float *out, void *workspace,
                        size_t workspace_bytes, cudaStream_t st) {
    const int rows = n_groups * rows_per_group, width = n_heads * kv->head_dim;
    if (int rc = attn_check(kv, n_heads, n_groups, rows, rows_per_group, max_blocks)) return rc;
    const AttnPlan p = attn_plan(kv, n_heads, n_groups, rows, rows_per_group, max_blocks);
    if (vxc_kv8_attn_workspace_bytes(kv, n_heads, n_groups, rows, rows_per_group, max_blocks) > workspace_bytes) {
        vxc_set_error("vxc_forward: attention workspace too small");
        return -4;
    }
    const Kv8AttnArgs a = {*kv, q, width, n_heads, scale, d_table, max_blocks, NULL, d_pos, d_seq, n_groups, rows,
                           rows_per_group, out, width, (float *)workspace};
    return attn_run(a, p, st);
}
