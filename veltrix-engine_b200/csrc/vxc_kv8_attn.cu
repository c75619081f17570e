// vxc_kv8_attn.cu — causal attention over the paged 8-bit KV cache
// (reference src/model.c:299-338, over its fp32 cache).
//   out_i,h = sum_j softmax_j(scale q_i,h . k_j) v_j,  j <= position of row i
#include "vxc_kv8.cuh"

#include <climits>

struct Kv8AttnArgs {
    vxc_kv8 kv;
    const float *q;
    long long ldq;
    int H;
    float scale;
    const int *table;
    int max_blocks;
    const int *row0;    // [n_req + 1]
    const int *pos;     // [n_req]
    int n_req, n_rows, max_new;
    float *out;
    long long ldo;
    unsigned int *err;
};

// One warp per (row, head), lanes over 32 tokens for the scores and over the
// head dim for the output; online softmax, all in fp32.
template <int TYPE, int HD>
__global__ void __launch_bounds__(128) k_kv8_attn_rows(const Kv8AttnArgs a) {
    __shared__ __align__(16) float qs[4][HD];
    pdl_trigger();
    pdl_wait();
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int i = blockIdx.x, h = blockIdx.y * 4 + w;
    if (i == 0 && h == 0 && lane == 0 && a.row0[a.n_req] > a.n_rows) vxc_flag_error(a.err, VXC_DERR_BAD_BLOCK);
    if (h >= a.H || i >= a.row0[a.n_req] || i >= a.n_rows) return;
    int lo = 0, hi = a.n_req;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.row0[mid] <= i) lo = mid; else hi = mid;
    }
    const int r = lo, t = i - a.row0[r], bs = a.kv.block_size, KH = a.kv.n_kv_heads, kvh = h / (a.H / KH);
    const long long last = (long long)a.pos[r] + t;   // last visible token
    if (t < 0 || t >= a.max_new || last >= (long long)a.max_blocks * bs) {
        if (lane == 0) vxc_flag_error(a.err, VXC_DERR_BAD_BLOCK);
        return;
    }
    const float *q = a.q + (size_t)i * a.ldq + (size_t)h * HD;
    for (int d = lane; d < HD; d += 32) qs[w][d] = q[d] * a.scale;
    __syncwarp();
    float m = -INFINITY, l = 0.0f, o[HD / 32];
    for (int d = 0; d < HD / 32; d++) o[d] = 0.0f;
    const uint8_t *kc = (const uint8_t *)a.kv.k, *vc = (const uint8_t *)a.kv.v;
    for (long long j0 = 0; j0 <= last; j0 += 32) {
        const long long j = j0 + lane;
        float s = -INFINITY, vs = 0.0f;
        size_t at = 0;
        if (j <= last) {
            const int b = a.table[(size_t)r * a.max_blocks + j / bs];
            if (b >= 0 && b < a.kv.n_blocks) {
                const size_t bh = (size_t)b * KH + kvh;
                at = (bh * bs + j % bs) * HD;
                vs = a.kv.v_scale[bh];
                float dot = 0.0f;
                for (int d = 0; d < HD; d++) dot = fmaf(qs[w][d], kv8_value<TYPE>(kc[at + d]), dot);
                s = dot * a.kv.k_scale[bh];
            } else {
                vxc_flag_error(a.err, VXC_DERR_BAD_BLOCK);
            }
        }
        const float mn = fmaxf(m, warp_max(s));
        if (mn == -INFINITY) continue;
        const float c = expf(m - mn), e = s == -INFINITY ? 0.0f : expf(s - mn);
        l = l * c + warp_sum(e);
        for (int d = 0; d < HD / 32; d++) o[d] *= c;
        m = mn;
        for (int jj = 0; jj < 32; jj++) {
            const float ej = __shfl_sync(0xffffffffu, e, jj) * __shfl_sync(0xffffffffu, vs, jj);
            const size_t aj = __shfl_sync(0xffffffffu, at, jj);
            if (ej == 0.0f) continue;
            for (int d = 0; d < HD / 32; d++) o[d] = fmaf(ej, kv8_value<TYPE>(vc[aj + d * 32 + lane]), o[d]);
        }
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    float *out = a.out + (size_t)i * a.ldo + (size_t)h * HD;
    for (int d = 0; d < HD / 32; d++) out[d * 32 + lane] = o[d] * inv;
}

typedef void (*attn_rows_t)(const Kv8AttnArgs);
template <int TYPE>
static attn_rows_t attn_rows_kernel(int hd) {
    switch (hd) {
        case 32: return k_kv8_attn_rows<TYPE, 32>;
        case 64: return k_kv8_attn_rows<TYPE, 64>;
        case 96: return k_kv8_attn_rows<TYPE, 96>;
        default: return k_kv8_attn_rows<TYPE, 128>;
    }
}

static int attn_check(const vxc_kv8 *kv, int n_heads, int n_req, int n_rows, int max_new, int max_blocks) {
    if (int rc = vxc_kv8_check(kv, "vxc_kv8_attn")) return rc;
    if (n_heads < 1 || n_heads > 65535 || n_heads % kv->n_kv_heads) {
        vxc_set_error("vxc_kv8_attn: %d heads over %d kv heads", n_heads, kv->n_kv_heads);
        return -4;
    }
    if (n_req < 1 || n_req > VXC_KV8_MAX_REQ || n_rows < 0 || n_rows > VXC_KV8_MAX_ROWS || max_new < 1 ||
        max_blocks < 1 || (long long)max_blocks * kv->block_size > INT_MAX) {
        vxc_set_error("vxc_kv8_attn: %d requests, %d rows (%d of one request), %d blocks per request", n_req, n_rows,
                      max_new, max_blocks);
        return -4;
    }
    return 0;
}

extern "C" size_t vxc_kv8_attn_workspace_bytes(const vxc_kv8 *kv, int n_heads, int n_req, int n_rows, int max_new,
                                               int max_blocks) {
    if (attn_check(kv, n_heads, n_req, n_rows, max_new, max_blocks)) return 0;
    return 0;
}

extern "C" int vxc_kv8_attn(const vxc_kv8 *kv, const float *q, long long ldq, int n_heads, float scale,
                            const int *d_table, int max_blocks, const int *d_row0, const int *d_pos, int n_req,
                            int n_rows, int max_new, float *out, long long ldo, void *workspace,
                            size_t workspace_bytes, void *stream) {
    if (int rc = attn_check(kv, n_heads, n_req, n_rows, max_new, max_blocks)) return rc;
    const long long width = (long long)n_heads * kv->head_dim;
    if (!d_table || !d_row0 || !d_pos ||
        (n_rows > 0 && (!q || !out || (uintptr_t)q % 16 || (uintptr_t)out % 16 || ldq < width || ldo < width ||
                        ldq % 4 || ldo % 4))) {
        vxc_set_error("vxc_kv8_attn: an array is missing or not aligned, or rows are shorter than %lld floats", width);
        return -4;
    }
    if (!(scale == scale) || scale - scale != 0.0f) {
        vxc_set_error("vxc_kv8_attn: scale is not finite");
        return -4;
    }
    if (int rc = vxc_require_device()) return rc;
    if (n_rows == 0) return 0;
    (void)workspace;
    (void)workspace_bytes;
    Kv8AttnArgs a = {*kv, q, ldq, n_heads, scale, d_table, max_blocks, d_row0, d_pos, n_req, n_rows, max_new, out, ldo,
                     vxc_device_error_ptr()};
    attn_rows_t f = kv->type == VXC_KV8_INT8 ? attn_rows_kernel<VXC_KV8_INT8>(kv->head_dim)
                                             : attn_rows_kernel<VXC_KV8_E4M3>(kv->head_dim);
    VXC_CUDA_OK(kv8_launch(f, dim3(n_rows, (n_heads + 3) / 4), dim3(128), 0, (cudaStream_t)stream, 1, a));
    return 0;
}
