// vxc_kv8.cu — the paged 8-bit KV cache: block tables and slot maps built
// from request lengths, and the append that quantises new K/V rows.
// (No reference counterpart: the reference keeps one contiguous fp32 cache,
// src/model.c:404-411.)
#include "vxc_kv8.cuh"
#include "vxc_smem_limit.h"

#include <climits>
#include <cooperative_groups.h>

namespace cg = cooperative_groups;

int vxc_kv8_check(const vxc_kv8 *kv, const char *who) {
    if (!kv) { vxc_set_error("%s: no cache", who); return -4; }
    if (kv->type != VXC_KV8_INT8 && kv->type != VXC_KV8_E4M3) {
        vxc_set_error("%s: cache type %d is neither VXC_KV8_INT8 nor VXC_KV8_E4M3", who, kv->type);
        return -4;
    }
    if (kv->block_size < 16 || kv->block_size > KV8_MAX_BS || kv->block_size % 16) {
        vxc_set_error("%s: block size %d is not a multiple of 16 from 16 to %d", who, kv->block_size, KV8_MAX_BS);
        return -4;
    }
    if (kv->head_dim != 32 && kv->head_dim != 64 && kv->head_dim != 96 && kv->head_dim != 128) {
        vxc_set_error("%s: head dim %d not supported (32, 64, 96 or 128)", who, kv->head_dim);
        return -4;
    }
    if (kv->n_kv_heads < 1 || kv->n_kv_heads > 65535) {
        vxc_set_error("%s: %d kv heads", who, kv->n_kv_heads);
        return -4;
    }
    if (kv->n_blocks < 1 || (long long)kv->n_blocks * kv->block_size > INT_MAX) {
        vxc_set_error("%s: %d blocks of %d tokens", who, kv->n_blocks, kv->block_size);
        return -4;
    }
    if (!kv->k || !kv->v || !kv->k_scale || !kv->v_scale || (uintptr_t)kv->k % 16 || (uintptr_t)kv->v % 16 ||
        (uintptr_t)kv->k_scale % 4 || (uintptr_t)kv->v_scale % 4) {
        vxc_set_error("%s: a cache array is missing or not aligned", who);
        return -4;
    }
    return 0;
}

namespace {
struct Runtime {   // for vxc_smem_allow
    typedef cudaError_t error;
    static constexpr cudaError_t ok = cudaSuccess;
    static cudaError_t device(int *d) { return cudaGetDevice(d); }
    static cudaError_t limit(const void *kernel, size_t *bytes) {
        cudaFuncAttributes fa;
        const cudaError_t e = cudaFuncGetAttributes(&fa, kernel);
        if (e == cudaSuccess) *bytes = (size_t)fa.maxDynamicSharedSizeBytes;
        return e;
    }
    static cudaError_t set_limit(const void *kernel, size_t bytes) {
        return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    }
};
}  // namespace

cudaError_t kv8_allow_smem(const void *kernel, size_t bytes) { return vxc_smem_allow<Runtime>(kernel, bytes); }

// ---------------------------------------------------------------------------
// block tables and slot maps
// ---------------------------------------------------------------------------
// One thread-block cluster (one CTA for few rows).  Every CTA scans the
// requests into shared memory: first row, first block taken and first block
// put back of each request.  After the cluster barrier every input that is
// rewritten has been read, and the CTAs share the outputs:
//  - block i taken: ring entry front + i; the request by a binary search of i
//    in the scan;
//  - block i put back: ring entry front + count + i.  held + count <=
//    n_blocks, so these entries are none of those taken from;
//  - slot of row i: the request by a binary search, then its table entry if
//    the request held the block before the call, else the ring entry it takes
//    (another CTA may not have written the table yet).
// Bound by latency: one pass over the lengths, a scan, one dependent load and
// a store per row.  Measured: 8 requests of one new token 4.5 us, 250 5.0 us;
// 32 prompts, 98 thousand rows, 12 us.
#define TB_THREADS 1024
#define TB_CLUSTER 8
#define TB_CLUSTER_ROWS 8192   // rows from which a cluster of TB_CLUSTER CTAs is used

// Index r with a[r] <= i < a[r + 1] (a ascending, a[0] = 0, i < a[n]).
__device__ __forceinline__ int tb_find(const int *a, int n, int i) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= i) lo = mid; else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(TB_THREADS)
    k_kv8_tables(const int *d_len, const int *d_new, int n, int bs, int nb, int max_blocks,
                 int *table, int *d_held, int *ring, int *state,
                 int n_rows, int *d_row0, int *d_slot, unsigned int *err) {
    extern __shared__ int sm[];
    int *row0 = sm, *pop0 = row0 + n + 1, *push0 = pop0 + n + 1;
    int *held = push0 + n + 1, *lens = held + n;   // [n]
    __shared__ int wsum[3][32], carry[3];
    __shared__ long long tot[4][32];
    __shared__ int wbad[32];
    const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
    pdl_trigger();
    pdl_wait();
    if (tid < 3) carry[tid] = 0;
    if (tid == 0) row0[0] = pop0[0] = push0[0] = 0;
    long long t_new = 0, t_held = 0, t_more = 0, t_less = 0;
    int bad = 0;
    __syncthreads();
    for (int c = 0; c < n; c += TB_THREADS) {
        const int r = c + tid;
        int x[3] = {0, 0, 0}, h = 0;
        if (r < n) {
            const int len = d_len[r], nw = d_new[r];
            h = d_held[r];
            if (len < 0 || nw < 0 || h < 0 || h > max_blocks) {
                bad |= 2;
            } else {
                const long long want = ((long long)len + nw + bs - 1) / bs;
                if (want > max_blocks) {
                    bad |= 1;
                } else {
                    x[0] = nw;
                    x[1] = (int)want > h ? (int)want - h : 0;
                    x[2] = (int)want < h ? h - (int)want : 0;
                    t_new += nw;
                    t_more += x[1];
                    t_less += x[2];
                    t_held += h;
                }
            }
            held[r] = h;
            lens[r] = len;
        }
        // inclusive scan of the three counts over the CTA (wrapping: totals are checked in 64 bits)
#pragma unroll
        for (int k = 0; k < 3; k++) {
            unsigned s = (unsigned)x[k];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned u = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += u;
            }
            x[k] = (int)s;
            if (lane == 31) wsum[k][w] = (int)s;
        }
        __syncthreads();
        if (w < 3) {
            unsigned s = (unsigned)wsum[w][lane];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned u = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += u;
            }
            const unsigned before = (unsigned)carry[w];
            const unsigned mine = (unsigned)wsum[w][lane];
            __syncwarp();
            wsum[w][lane] = (int)(before + s - mine);   // sum before this warp
            if (lane == 31) carry[w] = (int)(before + s);
        }
        __syncthreads();
        if (r < n) {
            row0[r + 1] = (int)((unsigned)x[0] + (unsigned)wsum[0][w]);
            pop0[r + 1] = (int)((unsigned)x[1] + (unsigned)wsum[1][w]);
            push0[r + 1] = (int)((unsigned)x[2] + (unsigned)wsum[2][w]);
        }
        __syncthreads();
    }
    {
        long long v[4] = {t_new, t_held, t_more, t_less};
#pragma unroll
        for (int k = 0; k < 4; k++) {
#pragma unroll
            for (int o = 16; o; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
            if (lane == 0) tot[k][w] = v[k];
        }
        bad = __reduce_or_sync(0xffffffffu, bad);
        if (lane == 0) wbad[w] = bad;
    }
    const int head = state[0], count = state[1];
    __syncthreads();
    {
        long long v[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            v[k] = tot[k][lane];
#pragma unroll
            for (int o = 16; o; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
        }
        t_new = v[0], t_held = v[1], t_more = v[2], t_less = v[3];
        bad = __reduce_or_sync(0xffffffffu, wbad[lane]);
    }
    if (head < 0 || head >= nb || count < 0 || t_held + count > nb || t_new > n_rows) bad |= 2;
    const int status = (bad & 2) ? 3 : (bad & 1) ? 2 : t_more > count ? 1 : 0;
    if (gridDim.x > 1) cg::this_cluster().sync();   // all inputs read; the outputs may change from here on
    const int gt = blockIdx.x * TB_THREADS + tid, gs = gridDim.x * TB_THREADS;
    if (status) {
        for (int i = gt; i <= n; i += gs) d_row0[i] = 0;
        for (int i = gt; d_slot && i < n_rows; i += gs) d_slot[i] = -1;
        if (gt == 0) {
            state[2] = status;
            if (status > 1) vxc_flag_error(err, VXC_DERR_BAD_BLOCK);
        }
        return;
    }
    for (int r = gt; r <= n; r += gs) {
        d_row0[r] = row0[r];
        if (r < n) d_held[r] = held[r] + (pop0[r + 1] - pop0[r]) - (push0[r + 1] - push0[r]);
    }
    auto ring_at = [&](long long i) -> int & {   // i <= n_blocks
        const long long at = head + i;
        return ring[at >= nb ? at - nb : at];
    };
    for (int i = gt; i < (int)t_more; i += gs) {
        const int r = tb_find(pop0, n, i), b = ring_at(i);
        table[(size_t)r * max_blocks + held[r] + (i - pop0[r])] = b;
        if (b < 0 || b >= nb) vxc_flag_error(err, VXC_DERR_BAD_BLOCK);
    }
    for (int i = gt; i < (int)t_less; i += gs) {
        const int r = tb_find(push0, n, i);
        int *e = table + (size_t)r * max_blocks + held[r] - (push0[r + 1] - i);
        ring_at((long long)count + i) = *e;
        *e = -1;
    }
    if (gt == 0) {
        state[0] = (int)((head + t_more) % nb);
        state[1] = (int)(count - t_more + t_less);
        state[2] = 0;
    }
    // four rows at a time, so that their loads are under way together
    const int total = (int)t_new;
    for (int i0 = gt; d_slot && i0 < n_rows; i0 += 4 * gs) {
        int b[4], off[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int i = i0 + k * gs;
            b[k] = off[k] = -1;
            if (i < total) {
                const int r = tb_find(row0, n, i);
                const unsigned p = (unsigned)lens[r] + (unsigned)(i - row0[r]);
                const int j = (int)(p / (unsigned)bs);
                off[k] = (int)(p - (unsigned)j * (unsigned)bs);
                b[k] = j < held[r] ? table[(size_t)r * max_blocks + j] : ring_at((long long)pop0[r] + j - held[r]);
            }
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int i = i0 + k * gs;
            if (i >= n_rows) break;
            const bool ok = b[k] >= 0 && b[k] < nb;
            if (!ok && i < total) vxc_flag_error(err, VXC_DERR_BAD_BLOCK);
            d_slot[i] = ok ? b[k] * bs + off[k] : -1;
        }
    }
}

extern "C" int vxc_kv8_tables(const int *d_len, const int *d_new, int n_req, int block_size, int n_blocks,
                              int max_blocks, int *d_table, int *d_held, int *d_free, int *d_state, int n_rows,
                              int *d_row0, int *d_slot, void *stream) {
    if (!d_len || !d_new || !d_table || !d_held || !d_free || !d_state || !d_row0 || (n_rows > 0 && !d_slot) ||
        !kv8_words(d_len, d_new, d_table, d_held, d_free, d_state, d_row0, d_slot)) {
        vxc_set_error("vxc_kv8_tables: an array is missing or not aligned");
        return -4;
    }
    if (n_req < 1 || n_req > VXC_KV8_MAX_REQ || n_rows < 0 || n_rows > KV8_MAX_TOKENS) {
        vxc_set_error("vxc_kv8_tables: %d requests (1 to %d), %d rows", n_req, VXC_KV8_MAX_REQ, n_rows);
        return -4;
    }
    if (block_size < 16 || block_size > KV8_MAX_BS || block_size % 16 || n_blocks < 1 || max_blocks < 1 ||
        (long long)n_blocks * block_size > INT_MAX || (long long)max_blocks * block_size > KV8_MAX_TOKENS) {
        vxc_set_error("vxc_kv8_tables: %d blocks of %d tokens, %d per request", n_blocks, block_size, max_blocks);
        return -4;
    }
    if (int rc = vxc_require_device()) return rc;
    const size_t smem = (size_t)(5 * n_req + 3) * sizeof(int);
    const int nc = n_rows >= TB_CLUSTER_ROWS ? TB_CLUSTER : 1;
    // the static arrays take the rest of the default 48 KB
    if (smem > 44 * 1024) VXC_CUDA_OK(kv8_allow_smem((const void *)k_kv8_tables, (5 * VXC_KV8_MAX_REQ + 3) * sizeof(int)));
    VXC_CUDA_OK(kv8_launch(k_kv8_tables, dim3(nc), dim3(TB_THREADS), smem, (cudaStream_t)stream, nc, d_len, d_new,
                           n_req, block_size, n_blocks, max_blocks, d_table, d_held, d_free, d_state, n_rows, d_row0,
                           d_slot, vxc_device_error_ptr()));
    return 0;
}

// The forward's form: no slot map, any number of rows (sizes checked when the
// sequence set was made).
int vxc_kv8_tables_only(const int *d_len, const int *d_new, int n_req, int block_size, int n_blocks, int max_blocks,
                        int *d_table, int *d_held, int *d_free, int *d_state, int *d_row0, cudaStream_t st) {
    const size_t smem = (size_t)(5 * n_req + 3) * sizeof(int);
    if (smem > 44 * 1024) VXC_CUDA_OK(kv8_allow_smem((const void *)k_kv8_tables, (5 * VXC_KV8_MAX_REQ + 3) * sizeof(int)));
    VXC_CUDA_OK(kv8_launch(k_kv8_tables, dim3(1), dim3(TB_THREADS), smem, st, 1, d_len, d_new, n_req, block_size, n_blocks,
                           max_blocks, d_table, d_held, d_free, d_state, INT_MAX, d_row0, (int *)NULL,
                           vxc_device_error_ptr()));
    return 0;
}

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
// A run = the rows of one block (they stand together in the slot map).  CTA =
// (window of rows, head, K or V), cut into teams of TS threads; each team goes
// over runs that begin in the window.  Two passes over a run's elements: their
// largest magnitude, then the codes; the first AP_HELD passes stay in registers
// in between, the rest is read again from L2.  TS is chosen so that a block's
// rows are AP_HELD passes, and the window so that a team has about one run: a
// CTA that finds no run costs a slot on its SM for the time of a load (with
// windows of 16 rows and blocks of 64 these took longer than the work).
// Bytes bound it: 4 read and 1 written per element.  Measured (heads of 128): 50
// thousand rows of 8 kv heads 100 us, 5.1 TB/s (windows of 16 rows and one team
// a CTA: 319 us); 32 requests of 7 rows 5.9 us; 8 rows of 32 kv heads 4.4 us.
#define AP_THREADS 256
#define AP_HELD 8

template <int TS>
__device__ __forceinline__ void team_sync(int team) {
    if (TS == 32) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(TS) : "memory");
}

template <int TYPE, int TS>
__global__ void __launch_bounds__(AP_THREADS, 4)
    k_kv8_append(const vxc_kv8 kv, const float *kx, long long ldk, const float *vx,
                 long long ldv, const int *slot, int n_rows, int window, int lsh, int units, unsigned int *err) {
    constexpr int TEAMS = AP_THREADS / TS;
    extern __shared__ int sm[];
    __shared__ float red[AP_THREADS / 32];
    __shared__ int n_lead;
    const int tid = threadIdx.x, lane = tid & 31, team = tid / TS, tt = tid % TS;
    const int bs = kv.block_size, hd = kv.head_dim, cap = kv.n_blocks * bs;
    // this CTA's parts of a row: K and V of head 0, K and V of head 1, ...
    const int parts = (2 * kv.n_kv_heads + units - 1) / units, u0 = (int)(blockIdx.x % (unsigned)parts) * units;
    const int u1 = min(u0 + units, 2 * kv.n_kv_heads);
    const int len = window + bs + 33;   // the row before the window, a run that begins with its last row, a warp's look behind it
    int *s_blk = sm, *s_off = s_blk + len, *lead = s_off + len, *win = lead + window + team * bs;
    pdl_trigger();
    pdl_wait();
    // blocks and offsets of the row before the window, its rows, and as many as a run may go on
    const int i0 = (int)(blockIdx.x / (unsigned)parts) * window;
    if (tid == 0) n_lead = 0;
    auto split = [&](int i, int &blk, int &off) {
        const int s = i >= 0 && i < n_rows ? slot[i] : -1;
        const bool ok = s >= 0 && s < cap;
        blk = ok ? s / bs : -1;
        off = ok ? s - blk * bs : 0;
        return s;
    };
    for (int t = tid; t < len; t += AP_THREADS) {
        const int s = split(i0 - 1 + t, s_blk[t], s_off[t]);
        if (s != -1 && s_blk[t] < 0 && u0 == 0 && t >= 1 && t <= window) vxc_flag_error(err, VXC_DERR_BAD_BLOCK);
    }
    __syncthreads();
    for (int t = tid; t < window; t += AP_THREADS)
        if (s_blk[t + 1] >= 0 && s_blk[t + 1] != s_blk[t]) lead[atomicAdd(&n_lead, 1)] = t;   // (runs in any order)
    __syncthreads();
    const int c = tt & ((1 << lsh) - 1), jr = tt >> lsh, rpp = TS >> lsh;   // float4 of a row, row of a pass, rows a pass
    const bool on = 4 * c < hd;
    bool odd = false;   // a NaN or infinity was stored as 0
    for (int k = team; k < n_lead; k += TEAMS) {
        const int t0 = lead[k] + 1, first = i0 + lead[k], blk = s_blk[t0];
        // a run goes on past the table only if it has slots twice
        auto blk_of = [&](int j) {
            if (t0 + j < len) return s_blk[t0 + j];
            int b, o;
            split(first + j, b, o);
            return b;
        };
        auto off_of = [&](int j) {
            if (t0 + j < len) return s_off[t0 + j];
            int b, o;
            split(first + j, b, o);
            return o;
        };
        // rows of the run; plain: their offsets ascend one by one, as from vxc_kv8_tables (then win is not needed)
        const int off0 = s_off[t0];
        int n = 0;
        bool plain = true;
#pragma unroll 1
        for (bool more = true; more;) {
            const bool mine = blk_of(n + lane) == blk;
            const unsigned in = __ballot_sync(0xffffffffu, mine);
            const unsigned up = __ballot_sync(0xffffffffu, off_of(n + lane) == off0 + n + lane);
            more = in == 0xffffffffu;
            const int k = more ? 32 : __ffs(~in) - 1;
            plain = plain && (~up & (more ? 0xffffffffu : (1u << k) - 1u)) == 0;
            n += k;
        }
        if (!plain) {
            team_sync<TS>(team);   // the last run's win is no longer read
            for (int t = tt; t < bs; t += TS) win[t] = -1;
            team_sync<TS>(team);
#pragma unroll 1
            for (int j = tt; j < n; j += TS) atomicMax(&win[off_of(j)], j);
            team_sync<TS>(team);
        }
        auto written = [&](int t) { return plain ? t >= off0 && t < off0 + n : win[t] >= 0; };
        // NaN and infinity count as 0
        auto finite = [](float4 f) {
            const float big = 3.402823466e38f;
            f.x = fabsf(f.x) <= big ? f.x : 0.0f;
            f.y = fabsf(f.y) <= big ? f.y : 0.0f;
            f.z = fabsf(f.z) <= big ? f.z : 0.0f;
            f.w = fabsf(f.w) <= big ? f.w : 0.0f;
            return f;
        };
        auto max4 = [](float4 f) { return fmaxf(fmaxf(fabsf(f.x), fabsf(f.y)), fmaxf(fabsf(f.z), fabsf(f.w))); };
        // 0, or NaN if one of the four is none or infinite
        auto nan4 = [](float4 f, float t) { return fmaf(f.x, 0.0f, fmaf(f.y, 0.0f, fmaf(f.z, 0.0f, fmaf(f.w, 0.0f, t)))); };
#pragma unroll 1
        for (int u = u0; u < u1; u++) {
            const int h = u >> 1, isv = u & 1;
            const size_t ld4 = (size_t)(isv ? ldv : ldk) / 4;
            const float4 *row = reinterpret_cast<const float4 *>((isv ? vx : kx) + (size_t)h * hd) + (size_t)first * ld4 + c;
            auto load = [&](int j) { return row[(size_t)j * ld4]; };
            float *sc = (isv ? kv.v_scale : kv.k_scale) + (size_t)blk * kv.n_kv_heads + h;
            const float held = *sc;
            float4 keep[AP_HELD];
            {
                const float4 *p = row + (size_t)jr * ld4;
                const size_t step = (size_t)rpp * ld4;
#pragma unroll
                for (int i = 0; i < AP_HELD; i++) {
                    keep[i] = on && jr + i * rpp < n ? *p : make_float4(0.f, 0.f, 0.f, 0.f);
                    p += step;
                }
            }
            team_sync<TS>(team);   // the last part's red is no longer read
            float mx = 0.0f, nan = 0.0f;
#pragma unroll
            for (int i = 0; i < AP_HELD; i++) nan = nan4(keep[i], nan);
#pragma unroll
            for (int i = 0; i < AP_HELD; i++) mx = fmaxf(mx, max4(keep[i]));
            // a thread with a NaN or an infinity reads its rows again, one by one
            const bool bad = nan != 0.0f;
            if (bad) {
                odd = true;
                mx = 0.0f;
            }
#pragma unroll 1
            for (int j = jr + (bad ? 0 : AP_HELD * rpp); on && j < n; j += rpp) {
                const float4 f = load(j);
                if (nan4(f, 0.0f) != 0.0f) odd = true;
                mx = fmaxf(mx, max4(finite(f)));
            }
            mx = warp_max(mx);
            if (TS > 32) {
                if (lane == 0) red[tid >> 5] = mx;
                team_sync<TS>(team);
#pragma unroll
                for (int i = 0; i < TS / 32; i++) mx = fmaxf(mx, red[team * (TS / 32) + i]);
            } else {
                __syncwarp();
            }
            const float old = written(0) ? 0.0f : held;
            const float s = fmaxf(old, mx > 0.0f ? __uint_as_float((uint32_t)(kv8_scale_exp(mx, TYPE) + 127) << 23) : 0.0f);
            uint8_t *dst = (uint8_t *)(isv ? kv.v : kv.k) + ((size_t)blk * kv.n_kv_heads + h) * bs * hd;
            if (s > old && old > 0.0f) {
                // the scale grew: the tokens that stay are rounded again
                const float ratio = old / s;
#pragma unroll 1
                for (int j = jr; on && j < bs; j += rpp) {
                    if (written(j)) continue;
                    uint32_t *p = reinterpret_cast<uint32_t *>(dst + (size_t)j * hd) + c;
                    const uint32_t q = *p;
                    *p = kv8_pack4<TYPE>(kv8_value<TYPE>(q & 0xFF) * ratio, kv8_value<TYPE>((q >> 8) & 0xFF) * ratio,
                                         kv8_value<TYPE>((q >> 16) & 0xFF) * ratio, kv8_value<TYPE>(q >> 24) * ratio);
                }
            }
            // dividing by a power of two is a product with its inverse; a scale that
            // is none (written by the caller) is divided by
            const bool pow2 = (__float_as_uint(s) & 0x7FFFFFu) == 0;
            const float inv = s > 0.0f ? 1.0f / s : 0.0f;
            auto store = [&](int off, float4 f) {
                uint32_t *to = reinterpret_cast<uint32_t *>(dst + (size_t)off * hd) + c;
                if (pow2 || s == 0.0f)
                    *to = TYPE == VXC_KV8_INT8 ? kv8_pack4_int8(f.x, f.y, f.z, f.w, inv)
                                               : kv8_pack4<TYPE>(f.x * inv, f.y * inv, f.z * inv, f.w * inv);
                else
                    *to = kv8_pack4<TYPE>(f.x / s, f.y / s, f.z / s, f.w / s);
            };
            int held_rows = 0;   // rows stored from registers
            if (plain && pow2 && !bad) {
                uint32_t *to = reinterpret_cast<uint32_t *>(dst + (off0 + jr) * hd) + c;
                const int step = rpp * hd / 4;
#pragma unroll
                for (int i = 0; i < AP_HELD; i++) {
                    if (on && jr + i * rpp < n)
                        to[i * step] =
                            TYPE == VXC_KV8_INT8 ? kv8_pack4_int8(keep[i].x, keep[i].y, keep[i].z, keep[i].w, inv)
                                                 : kv8_pack4<TYPE>(keep[i].x * inv, keep[i].y * inv, keep[i].z * inv, keep[i].w * inv);
                }
                held_rows = AP_HELD * rpp;
            }
#pragma unroll 1
            for (int j = jr + held_rows; on && j < n; j += rpp) {
                const int off = off_of(j);
                if (plain || win[off] == j) store(off, finite(load(j)));   // (not if a later row has this slot)
            }
            if (tt == 0 && s != held) *sc = s;
        }
    }
    if (__any_sync(0xffffffffu, odd) && lane == 0) vxc_flag_error(err, VXC_DERR_NONFINITE);
}

typedef void (*append_kernel_t)(const vxc_kv8, const float *, long long, const float *, long long, const int *, int,
                                int, int, int, unsigned int *);
template <int TYPE>
static append_kernel_t append_kernel(int ts) {
    switch (ts) {
        case 32: return k_kv8_append<TYPE, 32>;
        case 64: return k_kv8_append<TYPE, 64>;
        case 128: return k_kv8_append<TYPE, 128>;
        default: return k_kv8_append<TYPE, 256>;
    }
}

extern "C" int vxc_kv8_append(const vxc_kv8 *kv, const float *k, long long ldk, const float *v, long long ldv,
                              const int *d_slot, int n_rows, void *stream) {
    if (int rc = vxc_kv8_check(kv, "vxc_kv8_append")) return rc;
    if (n_rows < 0 || n_rows > VXC_KV8_MAX_ROWS) {
        vxc_set_error("vxc_kv8_append: %d rows (0 to %d)", n_rows, VXC_KV8_MAX_ROWS);
        return -4;
    }
    const long long width = (long long)kv->n_kv_heads * kv->head_dim;
    if (n_rows > 0 && (!k || !v || !d_slot || (uintptr_t)k % 16 || (uintptr_t)v % 16 || ldk < width || ldv < width ||
                       ldk % 4 || ldv % 4 || !kv8_words(d_slot))) {
        vxc_set_error("vxc_kv8_append: rows or slots missing or not aligned, or rows shorter than %lld floats", width);
        return -4;
    }
    if (int rc = vxc_require_device()) return rc;
    if (n_rows == 0) return 0;
    const int bs = kv->block_size, lsh = kv->head_dim == 32 ? 3 : kv->head_dim == 64 ? 4 : 5;
    // threads for a block's rows in AP_HELD passes
    int ts = 32;
    while (ts < AP_THREADS && (ts >> lsh) * AP_HELD < bs) ts *= 2;
    // rows per CTA: as many as keep two rounds of CTAs on the GPU (4 fit an SM), at most a block per
    // team: a step's few rows, each probably in a block of its own, go to as many CTAs
    const int most = AP_THREADS / ts * bs;
    const long long even = ((long long)n_rows * kv->n_kv_heads * 2 + 2 * 4 * 148 - 1) / (2 * 4 * 148);
    const int window = even < 1 ? 1 : even < most ? (int)even : most;
    // K and V of two heads per CTA when there are CTAs enough: a run is looked up once for them
    const int units = even >= 4ll * most ? 4 : 1;
    const size_t smem = (size_t)(2 * (window + bs + 33) + window + AP_THREADS / ts * bs) * sizeof(int);
    append_kernel_t f = kv->type == VXC_KV8_INT8 ? append_kernel<VXC_KV8_INT8>(ts) : append_kernel<VXC_KV8_E4M3>(ts);
    const long long grid = (long long)((n_rows + window - 1) / window) * ((2 * kv->n_kv_heads + units - 1) / units);
    if (grid > INT_MAX) {
        vxc_set_error("vxc_kv8_append: %d rows of %d heads", n_rows, kv->n_kv_heads);
        return -4;
    }
    VXC_CUDA_OK(kv8_launch(f, dim3((unsigned)grid), dim3(AP_THREADS), smem,
                           (cudaStream_t)stream, 1, *kv, k, ldk, v, ldv, d_slot, n_rows, window, lsh, units,
                           vxc_device_error_ptr()));
    return 0;
}
