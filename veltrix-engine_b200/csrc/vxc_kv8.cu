// vxc_kv8.cu — the paged 8-bit KV cache: block tables and slot maps built
// from request lengths, and the append that quantises new K/V rows.
// (No reference counterpart: the reference keeps one contiguous fp32 cache,
// src/model.c:404-411.)
#include "vxc_kv8.cuh"

#include <atomic>
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

// The limit is per kernel and device and only ever raised; a kernel that has
// it on a device is remembered, since asking costs a launch's time.
cudaError_t kv8_allow_smem(const void *kernel, size_t bytes) {
    if (bytes <= 48 * 1024) return cudaSuccess;
    struct Entry {
        std::atomic<const void *> kernel;
        std::atomic<size_t> bytes[64];
    };
    static Entry seen[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    Entry *own = nullptr;
    for (Entry &s : seen) {
        const void *k = s.kernel.load(std::memory_order_acquire);
        if (!k && s.kernel.compare_exchange_strong(k, kernel)) k = kernel;
        if (k == kernel) {
            own = &s;
            break;
        }
    }
    if (own && dev < 64 && own->bytes[dev].load(std::memory_order_acquire) >= bytes) return cudaSuccess;
    cudaFuncAttributes fa;
    e = cudaFuncGetAttributes(&fa, kernel);
    if (e == cudaSuccess && (size_t)fa.maxDynamicSharedSizeBytes < bytes)
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess && own && dev < 64) {
        size_t have = own->bytes[dev].load();
        while (have < bytes && !own->bytes[dev].compare_exchange_weak(have, bytes)) {}
    }
    return e;
}

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
// a store per row.
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
    k_kv8_tables(const int *__restrict__ d_len, const int *__restrict__ d_new, int n, int bs, int nb, int max_blocks,
                 int *__restrict__ table, int *__restrict__ d_held, int *__restrict__ ring, int *__restrict__ state,
                 int n_rows, int *__restrict__ d_row0, int *__restrict__ d_slot, unsigned int *err) {
    extern __shared__ int sm[];
    int *row0 = sm, *pop0 = row0 + n + 1, *push0 = pop0 + n + 1, *held = push0 + n + 1;   // held[n]
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
        for (int i = gt; i < n_rows; i += gs) d_slot[i] = -1;
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
    auto ring_at = [&](long long i) -> int & { return ring[(head + i) % nb]; };
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
    const int total = (int)t_new;
    for (int i = gt; i < n_rows; i += gs) {
        int s = -1;
        if (i < total) {
            const int r = tb_find(row0, n, i);
            const unsigned p = (unsigned)d_len[r] + (unsigned)(i - row0[r]);
            const int j = (int)(p / (unsigned)bs);
            const int b = j < held[r] ? table[(size_t)r * max_blocks + j] : ring_at((long long)pop0[r] + j - held[r]);
            if (b >= 0 && b < nb) s = b * bs + (int)(p % (unsigned)bs);
            else vxc_flag_error(err, VXC_DERR_BAD_BLOCK);
        }
        d_slot[i] = s;
    }
}

extern "C" int vxc_kv8_tables(const int *d_len, const int *d_new, int n_req, int block_size, int n_blocks,
                              int max_blocks, int *d_table, int *d_held, int *d_free, int *d_state, int n_rows,
                              int *d_row0, int *d_slot, void *stream) {
    if (!d_len || !d_new || !d_table || !d_held || !d_free || !d_state || !d_row0 || (n_rows > 0 && !d_slot)) {
        vxc_set_error("vxc_kv8_tables: an array is missing");
        return -4;
    }
    if (n_req < 1 || n_req > VXC_KV8_MAX_REQ || n_rows < 0) {
        vxc_set_error("vxc_kv8_tables: %d requests (1 to %d), %d rows", n_req, VXC_KV8_MAX_REQ, n_rows);
        return -4;
    }
    if (block_size < 16 || block_size > KV8_MAX_BS || block_size % 16 || n_blocks < 1 || max_blocks < 1 ||
        (long long)n_blocks * block_size > INT_MAX || (long long)max_blocks * block_size > KV8_MAX_TOKENS) {
        vxc_set_error("vxc_kv8_tables: %d blocks of %d tokens, %d per request", n_blocks, block_size, max_blocks);
        return -4;
    }
    if (int rc = vxc_require_device()) return rc;
    const size_t smem = (size_t)(4 * n_req + 3) * sizeof(int);
    const int nc = n_rows >= TB_CLUSTER_ROWS ? TB_CLUSTER : 1;
    // the static arrays take the rest of the default 48 KB
    if (smem > 44 * 1024) VXC_CUDA_OK(kv8_allow_smem((const void *)k_kv8_tables, (4 * VXC_KV8_MAX_REQ + 3) * sizeof(int)));
    VXC_CUDA_OK(kv8_launch(k_kv8_tables, dim3(nc), dim3(TB_THREADS), smem, (cudaStream_t)stream, nc, d_len, d_new,
                           n_req, block_size, n_blocks, max_blocks, d_table, d_held, d_free, d_state, n_rows, d_row0,
                           d_slot, vxc_device_error_ptr()));
    return 0;
}

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
// A run = the rows of one block (they stand together in the slot map); CTA =
// (window of rows, head, K or V) and goes over the runs that begin in its
// window.  Two passes over a run's elements: their largest magnitude, then the
// codes; the first AP_HELD float4 of each thread stay in registers in between
// (a block of 64 tokens x 128 elements whole), the rest is read again from L2.
// Bytes bound it: 4 read and 1 written per element.
#define AP_THREADS 256
#define AP_HELD 8

template <int TYPE, int HD>
__global__ void __launch_bounds__(AP_THREADS)
    k_kv8_append(const vxc_kv8 kv, const float *__restrict__ kx, long long ldk, const float *__restrict__ vx,
                 long long ldv, const int *__restrict__ slot, int n_rows, int window, unsigned int *err) {
    constexpr int C4 = HD / 4;   // float4 per row
    __shared__ int win[KV8_MAX_BS];
    __shared__ float red[AP_THREADS / 32];
    const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
    const int bs = kv.block_size, h = blockIdx.y, cap = kv.n_blocks * bs;
    const float *x = (blockIdx.z ? vx : kx) + (size_t)h * HD;
    const long long ld = blockIdx.z ? ldv : ldk;
    uint8_t *codes = (uint8_t *)(blockIdx.z ? kv.v : kv.k);
    float *scales = blockIdx.z ? kv.v_scale : kv.k_scale;
    pdl_trigger();
    pdl_wait();
    // rows of the window that begin a run
    const int i0 = blockIdx.x * window;
    unsigned leaders;
    {
        const int i = i0 + lane;
        bool lead = false;
        if (lane < window && i < n_rows) {
            const int s = slot[i], p = i ? slot[i - 1] : -1;
            if (s >= 0 && s < cap) lead = p < 0 || p / bs != s / bs;
            else if (s != -1 && h == 0 && w == 0) vxc_flag_error(err, VXC_DERR_BAD_BLOCK);
        }
        leaders = __ballot_sync(0xffffffffu, lead);
    }
    bool odd = false;   // a NaN or infinity was stored as 0
    while (leaders) {
        const int first = i0 + __ffs(leaders) - 1;
        leaders &= leaders - 1;
        const int blk = slot[first] / bs;
        int n = 0;
        for (bool more = true; more;) {
            const int i = first + n + lane;
            const int s = i < n_rows ? slot[i] : -1;
            const unsigned in = __ballot_sync(0xffffffffu, s >= 0 && s / bs == blk);
            more = in == 0xffffffffu;
            n += more ? 32 : __ffs(~in) - 1;
        }
        __syncthreads();   // the last run's win and red are no longer read
        for (int t = tid; t < bs; t += AP_THREADS) win[t] = -1;
        __syncthreads();
        for (int j = tid; j < n; j += AP_THREADS) atomicMax(&win[slot[first + j] % bs], j);
        const int nu = n * C4;
        auto load = [&](int u) {
            float4 f = *reinterpret_cast<const float4 *>(x + (size_t)(first + u / C4) * ld + (size_t)(u % C4) * 4);
            const float big = 3.402823466e38f;
            if (!(fabsf(f.x) <= big)) { f.x = 0.0f; odd = true; }
            if (!(fabsf(f.y) <= big)) { f.y = 0.0f; odd = true; }
            if (!(fabsf(f.z) <= big)) { f.z = 0.0f; odd = true; }
            if (!(fabsf(f.w) <= big)) { f.w = 0.0f; odd = true; }
            return f;
        };
        auto max4 = [](float4 f) { return fmaxf(fmaxf(fabsf(f.x), fabsf(f.y)), fmaxf(fabsf(f.z), fabsf(f.w))); };
        float4 keep[AP_HELD];
        float mx = 0.0f;
#pragma unroll
        for (int i = 0; i < AP_HELD; i++) {
            const int u = tid + i * AP_THREADS;
            if (u < nu) {
                keep[i] = load(u);
                mx = fmaxf(mx, max4(keep[i]));
            }
        }
        for (int u = tid + AP_HELD * AP_THREADS; u < nu; u += AP_THREADS) mx = fmaxf(mx, max4(load(u)));
        mx = warp_max(mx);
        if (lane == 0) red[w] = mx;
        float *sc = scales + (size_t)blk * kv.n_kv_heads + h;
        const float held = *sc;
        __syncthreads();
        mx = red[0];
#pragma unroll
        for (int i = 1; i < AP_THREADS / 32; i++) mx = fmaxf(mx, red[i]);
        const float old = win[0] >= 0 ? 0.0f : held;
        const float s = fmaxf(old, mx > 0.0f ? __uint_as_float((uint32_t)(kv8_scale_exp(mx, TYPE) + 127) << 23) : 0.0f);
        uint8_t *dst = codes + ((size_t)blk * kv.n_kv_heads + h) * bs * HD;
        if (s > old && old > 0.0f) {
            // the scale grew: the tokens that stay are rounded again
            const float ratio = old / s;
            for (int u = tid; u < bs * HD / 4; u += AP_THREADS) {
                if (win[u / C4] >= 0) continue;
                uint32_t *p = reinterpret_cast<uint32_t *>(dst) + u;
                const uint32_t q = *p;
                *p = kv8_pack4<TYPE>(kv8_value<TYPE>(q & 0xFF) * ratio, kv8_value<TYPE>((q >> 8) & 0xFF) * ratio,
                                     kv8_value<TYPE>((q >> 16) & 0xFF) * ratio, kv8_value<TYPE>(q >> 24) * ratio);
            }
        }
        // dividing by a power of two is a product with its inverse; a scale that
        // is none (written by the caller) is divided by
        const bool pow2 = (__float_as_uint(s) & 0x7FFFFFu) == 0;
        const float inv = s > 0.0f ? 1.0f / s : 0.0f;
        auto store = [&](int u, float4 f) {
            const int j = u / C4, off = slot[first + j] % bs;
            if (win[off] != j) return;   // a later row has this slot
            if (pow2 || s == 0.0f) {
                f.x *= inv, f.y *= inv, f.z *= inv, f.w *= inv;
            } else {
                f.x /= s, f.y /= s, f.z /= s, f.w /= s;
            }
            *reinterpret_cast<uint32_t *>(dst + (size_t)off * HD + (size_t)(u % C4) * 4) = kv8_pack4<TYPE>(f.x, f.y, f.z, f.w);
        };
#pragma unroll
        for (int i = 0; i < AP_HELD; i++) {
            const int u = tid + i * AP_THREADS;
            if (u < nu) store(u, keep[i]);
        }
        for (int u = tid + AP_HELD * AP_THREADS; u < nu; u += AP_THREADS) store(u, load(u));
        if (tid == 0 && s != held) *sc = s;
    }
    if (__any_sync(0xffffffffu, odd) && lane == 0) vxc_flag_error(err, VXC_DERR_NONFINITE);
}

typedef void (*append_kernel_t)(const vxc_kv8, const float *, long long, const float *, long long, const int *, int,
                                int, unsigned int *);
template <int TYPE>
static append_kernel_t append_kernel(int hd) {
    switch (hd) {
        case 32: return k_kv8_append<TYPE, 32>;
        case 64: return k_kv8_append<TYPE, 64>;
        case 96: return k_kv8_append<TYPE, 96>;
        default: return k_kv8_append<TYPE, 128>;
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
                       ldk % 4 || ldv % 4)) {
        vxc_set_error("vxc_kv8_append: rows missing, not 16-byte aligned, or shorter than %lld floats", width);
        return -4;
    }
    if (int rc = vxc_require_device()) return rc;
    if (n_rows == 0) return 0;
    // One row per CTA while all CTAs then fit the GPU at once or nearly so (a
    // decode or verify step); else 16, the shortest run of whole blocks.
    const int window = n_rows <= 512 ? 1 : 16;
    append_kernel_t f = kv->type == VXC_KV8_INT8 ? append_kernel<VXC_KV8_INT8>(kv->head_dim)
                                                 : append_kernel<VXC_KV8_E4M3>(kv->head_dim);
    VXC_CUDA_OK(kv8_launch(f, dim3((n_rows + window - 1) / window, kv->n_kv_heads, 2), dim3(AP_THREADS), 0,
                           (cudaStream_t)stream, 1, *kv, k, ldk, v, ldv, d_slot, n_rows, window,
                           vxc_device_error_ptr()));
    return 0;
}
