// vxc_kv8_attn.cuh — what the attention kernels over the paged 8-bit KV cache
// share: their arguments, a request's bounds, and the arithmetic of codes,
// queries and weights.
#pragma once
#include <limits.h>
#include "vxc_kv8.cuh"

struct Kv8AttnArgs {
    vxc_kv8 kv;
    const float *q;
    long long ldq;
    int H;
    float scale;
    const int *table;
    int max_blocks;
    const int *row0;    // [n_req + 1], or NULL: max_new rows each
    const int *pos;     // [n_req]
    const int *seq;     // NULL, or the table row of each request (negative: the request has no rows)
    int n_req, n_rows, max_new;
    float *out;
    long long ldo;
    float *part;        // records of the splits
    int S, sl_min;      // splits per request at most, tokens per split at least
    int pages;          // blocks a split may touch, rounded up to 4 (k_kv8_attn_few)
    int chunks;         // k_kv8_attn_few: CTAs with their own queries per request, kv head and split (then S is 1)
    int ranked;         // requests begin by length, longest first (at most KV8_RANKED)
    unsigned int *err;
};

#define KV8_HEAD 10.0f   // weights up to 2^(10 + 5): in fp16's range with 2^-34 of the largest as last place
#define KV8_LAG 5.0f
// The weights' reference is kept within 2^KV8_FLOOR of the largest softmax weight: 2^(m - mv + KV8_HEAD)
// and its inverse are then normal floats whatever V's scales are.  Where the floor holds, all that V adds is
// below 2^-115 of the softmax, and weights of a scale of 2^-126 still stand at 2^-1 (24 bits above the last place).
#define KV8_FLOOR 115.0f

// Weights are w = 2^(s - ref) c, c = v_scale * cv, cv = 2^(m - mv + KV8_HEAD), and the softmax's sum adds
// 2^(s - ref) * kv8_unit(..); ref is m on entry.  A visible token's w is at most 2^(KV8_HEAD + KV8_LAG), so
// with a c over 2^126 (vmax: the largest v_scale in sight) the weight that goes with it has 2^(s - m) below
// 2^-111, and with one over 2^128 may still be above 2^-126: exponentials are then taken 2^16 times
// as large, c and the unit 2^-16 times.
__device__ __forceinline__ float kv8_unit(float vmax, float &cv, float &ref) {
    if (vmax * cv <= 0x1p126f) return 1.0f;
    ref -= 16.0f;
    cv *= 0x1p-16f;
    return 0x1p-16f;
}
// What is over 2^127 even so belongs to weights below 2^-128 or to masked tokens: c stays finite, so that 0
// times it is 0.
__device__ __forceinline__ float kv8_factor(float v_scale, float cv) { return fminf(v_scale * cv, 0x1p127f); }

template <int N>
__device__ __forceinline__ void cp_async_zfill(uint32_t dst, const void *src, bool have) {
    const int n = have ? N : 0;
    if (N == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(n) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_async(uint32_t dst, const void *src) {
    if (N == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(N) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Shared memory to global, 16-byte aligned; returns when it is done.
__device__ __forceinline__ void bulk_s2g(void *dst, uint32_t src, uint32_t bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
    asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group 0;" ::: "memory");
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// a, b -> half2 of their fp16 roundings, and half2 of what is left
__device__ __forceinline__ uint32_t split_h2(float a, float b, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
    lo = *reinterpret_cast<const uint32_t *>(&l);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Four codes -> two half2, bytes (0, 1) and (2, 3).  int8: the byte with its
// sign bit flipped is the low byte of the half 1024 + 128 + code.
template <int TYPE>
__device__ __forceinline__ void codes_h2(uint32_t w, uint32_t &h01, uint32_t &h23) {
    if (TYPE == VXC_KV8_INT8) {
        const uint32_t x = w ^ 0x80808080u;
        uint32_t a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342);
        const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
        const __half2 ha = __hsub2(*reinterpret_cast<__half2 *>(&a), bias), hb = __hsub2(*reinterpret_cast<__half2 *>(&b), bias);
        h01 = *reinterpret_cast<const uint32_t *>(&ha);
        h23 = *reinterpret_cast<const uint32_t *>(&hb);
    } else {
        h01 = kv8_e4m3x2_h2((uint16_t)(w & 0xFFFFu));
        h23 = kv8_e4m3x2_h2((uint16_t)(w >> 16));
    }
}

// A power of two 2^k over l >= 1 and at most twice as large, and its inverse; 0 gives 2^-126 and 2^126.  (l is at most
// 2^36; NaN gives finite numbers.)
__device__ __forceinline__ float kv8_pow2_over(float l) { return __uint_as_float((__float_as_uint(l) & 0x7F800000u) + 0x00800000u); }
__device__ __forceinline__ float kv8_pow2_under(float l) { return __uint_as_float(0x7E800000u - (__float_as_uint(l) & 0x7F800000u)); }

// A request's rows and tokens as the call's arguments and arrays allow them.
struct Kv8Req {
    const int *table;
    int row0, T;     // first row; rows (clamped to n_rows, max_new and the table)
    int pos;         // position of the first row
    int kvlen;       // tokens the last row sees (0: none)
    bool over;       // something was clamped
};
__device__ __forceinline__ int kv8_row0(const Kv8AttnArgs &a, int r) { return a.row0 ? a.row0[r] : r * a.max_new; }
// table row s (none if negative), first row r0, end r1, position pos
__device__ __forceinline__ Kv8Req kv8_req_of(const Kv8AttnArgs &a, int s, int r0, int r1, int pos) {
    Kv8Req q;
    if (s < 0) r1 = r0;
    q.table = a.table + (size_t)max(s, 0) * a.max_blocks;
    q.pos = pos;
    q.row0 = max(r0, 0);
    long long T = (long long)r1 - r0;
    const long long cap = (long long)a.max_blocks * a.kv.block_size;
    const long long most = min(min((long long)a.max_new, (long long)a.n_rows - q.row0), cap - q.pos);
    q.over = r0 < 0 || (T > 0 && T > most);
    T = r0 < 0 ? 0 : min(T, most);
    q.T = (int)max(T, 0ll);
    q.kvlen = q.T > 0 ? max(q.pos + q.T, 0) : 0;
    return q;
}
__device__ __forceinline__ Kv8Req kv8_req(const Kv8AttnArgs &a, int r) {
    return kv8_req_of(a, a.seq ? a.seq[r] : r, kv8_row0(a, r), kv8_row0(a, r + 1), a.pos[r]);
}

// Requests begin longest first where not all CTAs fit the GPU at once, so that what begins last is short.
// (33 requests of one row behind up to 16384 tokens: 124 -> 100 us; 32 of 7 rows behind up to 4096:
// 122 -> 112 us.)  The position is length enough.
#define KV8_RANKED 128
// The request whose position is the k-th largest.  Called by the block's first KV8_RANKED threads (one
// warp with four requests a lane took 4 us for 43 of them); pos_s: KV8_RANKED + 1 ints of shared memory,
// 16-byte aligned.
__device__ __forceinline__ int kv8_ranked(const Kv8AttnArgs &a, int k, int *pos_s) {
    auto sync = [] { asm volatile("bar.sync 3, %0;" ::"n"(KV8_RANKED) : "memory"); };
    const int me = threadIdx.x, n = a.n_req, key = me < n ? a.pos[me] : INT_MIN;
    pos_s[me] = key;
    sync();
    if (me < n) {
        int rank = 0;
        auto count = [&](int p, int o) { rank += p > key || (p == key && o < me); };
        for (int o = 0; o < n; o += 4) {   // (INT_MIN behind the last: counts for no request)
            const int4 p = *reinterpret_cast<const int4 *>(pos_s + o);
            count(p.x, o), count(p.y, o + 1), count(p.z, o + 2), count(p.w, o + 3);
        }
        if (rank == k) pos_s[KV8_RANKED] = me;
    }
    sync();
    return pos_s[KV8_RANKED];
}

// Splits of a request: enough for SL_min tokens each, at most S.
__device__ __forceinline__ int kv8_splits(int kvlen, int sl_min, int S, int &SL) {
    const int want = min(max((kvlen + sl_min - 1) / sl_min, 1), S);
    SL = ((kvlen + want - 1) / want + 127) & ~127;
    return SL > 0 ? (kvlen + SL - 1) / SL : 1;
}

// Many queries per kv head (vxc_kv8_attn_many.cu): launch over at most `tiles`
// tiles of tile_q (32, 64 or 128) queries.
cudaError_t kv8_attn_many(const Kv8AttnArgs &a, int tile_q, int tiles, cudaStream_t st);
