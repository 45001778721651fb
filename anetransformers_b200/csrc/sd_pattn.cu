// sd_pattn.cu -- attention over a paged K/V cache: grouped heads, a prefix shared by every request of the batch,
// tanh-capped and distance-biased scores, windows.
//
//   o_t = sum_j p_j v_j / sum_j p_j,  p_j = exp(z_j - max z),
//   z_j = f(scale q_t.k_j) - slope (pos_t - pos_j),  f(s) = cap tanh(s / cap) or s
// over the visible j: prefix positions, then the request's own positions up to the row's, less those at a distance
// of `window` or more.
#include <cuda_bf16.h>

#include <algorithm>

#include "sd_common.cuh"
#include "sd_host.h"
#include "sd_paged.h"

using namespace sd;

namespace sd {
namespace {

__device__ __forceinline__ float pa_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float pa_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T> __device__ __forceinline__ T pa_from(float x);
template <> __device__ __forceinline__ __half pa_from<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 pa_from<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Request of a token: the last b with q_start[b] <= tok, or -1 if tok is none of its new tokens.  kv and q are cut
// to what the call allows.
struct TokReq {
    int b, t, kv, q;
};
__device__ __forceinline__ TokReq token_request(const sd_attn_args& a, int tok) {
    int lo = 0, hi = a.n_req;
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (a.q_start[m] <= tok) lo = m; else hi = m;
    }
    TokReq r{lo, tok - a.q_start[lo], 0, 0};
    r.q = min(max(a.q_len[lo], 0), a.max_q);
    r.kv = min(max(a.kv_len[lo], 0), a.max_kv);
    if (r.t < 0 || r.t >= r.q) r.b = -1;
    return r;
}

// One warp per (token, head), one key at a time: any head_dim, any strides.
template <class T>
__global__ void __launch_bounds__(128) k_pattn_general(const sd_attn_args a, int* err) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * 4 + warp;
    const int tok = (int)(row / a.n_heads), head = (int)(row - (long long)tok * a.n_heads);
    if (tok >= a.n_tokens) return;
    const TokReq rq = token_request(a, tok);
    if (lane == 0 && head == 0 && rq.b >= 0 && rq.t == 0 && (a.kv_len[rq.b] > a.max_kv || a.q_len[rq.b] > a.max_q))
        set_dev_error(err, DEV_ERR_BAD_ARG);
    if (rq.b < 0) return;
    const int hd = a.pool.head_dim, kvh = head / (a.n_heads / a.pool.n_kv_heads), ps = a.pool.page_size;
    const T* q = static_cast<const T*>(a.q) + (size_t)tok * a.q_ld + (size_t)head * a.q_head;
    T* out = static_cast<T*>(a.out) + (size_t)tok * a.out_ld + (size_t)head * a.out_head;
    const int own_i = rq.kv - rq.q + rq.t;
    float qv[8], acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        qv[i] = lane + 32 * i < hd ? pa_f32(q[lane + 32 * i]) : 0.f;
        acc[i] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    const float slope = a.alibi ? a.alibi[head] : 0.f;
    const int pos = a.prefix_len + own_i;
    const int first = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    for (int p = first; own_i >= 0 && p <= pos; ++p) {
        const int o = p - a.prefix_len;
        const int page = o < 0 ? a.prefix_table[p / ps] : a.table[(size_t)rq.b * a.table_ld + o / ps];
        if (page < 0 || page >= a.pool.n_pages) {
            if (lane == 0) set_dev_error(err, DEV_ERR_BAD_ARG);
            continue;
        }
        const size_t at = (size_t)page * a.pool.page_stride + (size_t)((o < 0 ? p : o) % ps) * a.pool.pos_stride +
                          (size_t)kvh * a.pool.head_stride;
        const T* k = static_cast<const T*>(a.pool.k) + at;
        const T* v = static_cast<const T*>(a.pool.v) + at;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (lane + 32 * i < hd) s = fmaf(qv[i], pa_f32(k[lane + 32 * i]), s);
        s = warp_sum(s) * a.scale;
        if (a.softcap > 0.f) s = a.softcap * tanhf(s / a.softcap);
        s -= slope * (float)(pos - p);
        const float mn = fmaxf(m, s), c = m == -INFINITY ? 0.f : expf(m - mn), w = expf(s - mn);
        m = mn;
        l = l * c + w;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (lane + 32 * i < hd) acc[i] = acc[i] * c + w * pa_f32(v[lane + 32 * i]);
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (lane + 32 * i < hd) out[lane + 32 * i] = pa_from<T>(acc[i] * inv);
}

int check_attention(const sd_attn_args* a) {
    const char* what = "sd_attention_dev";
    if (!a) return fail(SD_ERR_INVALID, "%s: null arguments", what);
    int rc = check_kv_pool(&a->pool, what);
    if (rc) return rc;
    if (!a->q || !a->out || !a->table || !a->kv_len || !a->q_start || !a->q_len)
        return fail(SD_ERR_INVALID, "%s: null argument", what);
    if (a->n_req < 1 || a->n_req > SD_PAGES_MAX_REQ)
        return fail(SD_ERR_INVALID, "%s: n_req %d outside 1..%d", what, a->n_req, SD_PAGES_MAX_REQ);
    if (a->n_heads < 1 || a->n_heads % a->pool.n_kv_heads || a->n_heads / a->pool.n_kv_heads > 128)
        return fail(SD_ERR_INVALID, "%s: %d heads over %d kv heads", what, a->n_heads, a->pool.n_kv_heads);
    if (a->n_tokens < 0 || a->max_q < 0 || a->max_kv < 0 || a->prefix_len < 0 || a->window < 0)
        return fail(SD_ERR_INVALID, "%s: negative size", what);
    if (a->table_ld < 1 || (int64_t)a->table_ld * a->pool.page_size < a->max_kv)
        return fail(SD_ERR_INVALID, "%s: max_kv %d beyond the block table (%d pages of %d)", what, a->max_kv, a->table_ld,
                    a->pool.page_size);
    if ((int64_t)a->prefix_len + a->max_kv > INT32_MAX - 1024) return fail(SD_ERR_INVALID, "%s: prefix too long", what);
    if (a->prefix_len > 0 && !a->prefix_table) return fail(SD_ERR_INVALID, "%s: a prefix needs its table", what);
    if (!(a->softcap >= 0.f) || !(a->scale == a->scale) || a->softcap > 1e30f)
        return fail(SD_ERR_INVALID, "%s: scale %g, softcap %g", what, a->scale, a->softcap);
    if (a->q_head < a->pool.head_dim || a->out_head < a->pool.head_dim || a->q_ld < 0 || a->out_ld < 0)
        return fail(SD_ERR_INVALID, "%s: strides", what);
    return SD_OK;
}

}  // namespace
}  // namespace sd

extern "C" {

size_t sd_attention_workspace(const sd_attn_args*) { return 0; }

int sd_attention_dev(const sd_attn_args* a, void* stream) {
    clear_error();
    int rc = check_attention(a), dev;
    if (rc) return rc;
    if (a->n_tokens == 0) return SD_OK;
    if ((rc = paged_device(a->pool.k, "sd_attention_dev", &dev))) return rc;
    const long long rows = (long long)a->n_tokens * a->n_heads;
    if ((rows + 3) / 4 > INT32_MAX) return fail(SD_ERR_INVALID, "sd_attention_dev: too many rows");
    const int grid = (int)((rows + 3) / 4);
    if (a->pool.dtype == SD_F16)
        k_pattn_general<__half><<<grid, 128, 0, (cudaStream_t)stream>>>(*a, device_error_word(dev));
    else
        k_pattn_general<__nv_bfloat16><<<grid, 128, 0, (cudaStream_t)stream>>>(*a, device_error_word(dev));
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? SD_OK : cuda_fail(e, "attention");
}

}  // extern "C"
