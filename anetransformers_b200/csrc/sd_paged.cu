// sd_paged.cu -- pages of a K/V cache shared by many requests: block tables and slot maps from request lengths,
// and K/V rows written through the slot map.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>

#include "sd_common.cuh"
#include "sd_host.h"
#include "sd_paged.h"

namespace cg = cooperative_groups;
using namespace sd;

namespace sd {

int check_pages(const sd_pages* p, const char* what) {
    if (!p || !p->table || !p->held || !p->free_pages || !p->n_free) return fail(SD_ERR_INVALID, "%s: null argument", what);
    if (p->n_req < 1 || p->n_req > SD_PAGES_MAX_REQ)
        return fail(SD_ERR_INVALID, "%s: n_req %d outside 1..%d", what, p->n_req, SD_PAGES_MAX_REQ);
    if (p->page_size < SD_PAGE_MIN || p->page_size > SD_PAGE_MAX || (p->page_size & (p->page_size - 1)))
        return fail(SD_ERR_INVALID, "%s: page_size %d is not a power of two in %d..%d", what, p->page_size, SD_PAGE_MIN, SD_PAGE_MAX);
    if (p->table_ld < 1 || (int64_t)p->table_ld * p->page_size > INT32_MAX || (int64_t)p->table_ld * p->n_req > INT32_MAX)
        return fail(SD_ERR_INVALID, "%s: table_ld %d", what, p->table_ld);
    if (p->n_pages < 1 || (int64_t)p->n_pages * p->page_size > INT32_MAX)
        return fail(SD_ERR_INVALID, "%s: n_pages %d", what, p->n_pages);
    return SD_OK;
}

int check_kv_pool(const sd_kv_pool* p, const char* what) {
    if (!p || !p->k || !p->v) return fail(SD_ERR_INVALID, "%s: null pool", what);
    if (p->page_size < SD_PAGE_MIN || p->page_size > SD_PAGE_MAX || (p->page_size & (p->page_size - 1)))
        return fail(SD_ERR_INVALID, "%s: page_size %d is not a power of two in %d..%d", what, p->page_size, SD_PAGE_MIN, SD_PAGE_MAX);
    if (p->n_pages < 1 || (int64_t)p->n_pages * p->page_size > INT32_MAX)
        return fail(SD_ERR_INVALID, "%s: n_pages %d", what, p->n_pages);
    if (p->n_kv_heads < 1 || p->n_kv_heads > 1024 || p->head_dim < 8 || p->head_dim > 256 || p->head_dim % 8)
        return fail(SD_ERR_INVALID, "%s: %d heads of %d", what, p->n_kv_heads, p->head_dim);
    if (p->dtype != SD_F16 && p->dtype != SD_BF16) return fail(SD_ERR_INVALID, "%s: pool dtype %d", what, p->dtype);
    if (p->page_stride < 1 || p->pos_stride < 1 || p->head_stride < p->head_dim)
        return fail(SD_ERR_INVALID, "%s: pool strides", what);
    return SD_OK;
}

int paged_device(const void* p, const char* what, int* dev) {
    int cur = -1;
    cudaError_t e = cudaGetDevice(&cur);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(SD_ERR_NO_DEVICE, "%s: %s", what, cudaGetErrorString(e));
    }
    cudaPointerAttributes at{};
    if ((e = cudaPointerGetAttributes(&at, p)) != cudaSuccess) return cuda_fail(e, what);
    if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged)
        return fail(SD_ERR_INVALID, "%s: not device memory", what);
    if (at.type == cudaMemoryTypeDevice && at.device != cur)
        return fail(SD_ERR_INVALID, "%s: the current device is %d but the arrays live on device %d", what, cur, at.device);
    *dev = cur;
    return SD_OK;
}

namespace {

// ---------------------------------------------------------------------------------------------
// Page plan.  All of a step is three prefix sums over the requests (surplus pages, wanted pages, new tokens) and
// three scatters.  Latency bound: a step moves a few bytes per request and token, so everything is one launch of one
// cluster.  Every CTA of the cluster computes the sums for itself (cheaper than handing them over), then the
// scatters are dealt over the cluster's threads, each finding its request by bisection in shared memory.  Cluster
// barriers separate reading the old state, pushing, taking and reading the new table; a step that moves no page
// passes none.  In a CUDA graph, one request and token takes 4.5 us; 256 requests, 1280 tokens 10.4 us (one CTA instead of
// the cluster took 23 us when the cluster took 9.3); 64 prompts replaced by 64 others, 36 thousand tokens, 16.6 us (59
// against 15).
// ---------------------------------------------------------------------------------------------
constexpr int kPlanThreads = 512;

constexpr size_t plan_smem(int n_req) { return ((size_t)4 * n_req + 3) * sizeof(int); }

struct PlanArgs {
    int32_t *table, *held, *free_pages, *n_free;
    int n_req, table_ld, n_pages, page_size;
    const int32_t *kv_len, *q_len;
    int q_stride, pos0, n_tokens;
    int32_t *q_start, *slots, *positions, *missing;
    int* err;
};

// Sum of two that are not negative; of tokens at most INT32_MAX (so that sums of lengths out of range still ascend; those of
// pages stay below it by the sizes that a plan takes).
__device__ __forceinline__ int plan_add(bool tokens, int x, int y) {
    return tokens ? (int)min((unsigned)x + (unsigned)y, (unsigned)INT32_MAX) : x + y;
}

// Last b in [0, n) with start[b] <= k (start ascends, start[0] = 0).
__device__ __forceinline__ int owner(const int* start, int n, int k) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (start[m] <= k) lo = m; else hi = m;
    }
    return lo;
}

__global__ void __launch_bounds__(kPlanThreads) k_pages_plan(const PlanArgs a) {
    extern __shared__ int sm[];
    __shared__ int wsum[3][kPlanThreads / 32];
    const int n = a.n_req, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int* back = sm;               // [n + 1] exclusive sums of surplus pages
    int* want = back + n + 1;     // of wanted pages
    int* toks = want + n + 1;     // of new tokens
    int* base = toks + n + 1;     // [n] first page that is given back or taken: min(held, needed)
    const cg::cluster_group cluster = cg::this_cluster();
    const int gtid = (int)cluster.block_rank() * kPlanThreads + tid, gn = (int)cluster.num_blocks() * kPlanThreads;
    const int cap = a.table_ld * a.page_size;
    const int free0 = *a.n_free;

    // sums: each thread takes `per` consecutive requests
    const int per = (n + kPlanThreads - 1) / kPlanThreads;
    const int b0 = min(n, tid * per), b1 = min(n, b0 + per);
    int s[3] = {0, 0, 0};
    bool bad = false;
    for (int b = b0; b < b1; ++b) {
        int kv = a.kv_len[b], q = a.q_len[b];
        if (kv < 0 || kv > cap) bad = true, kv = min(max(kv, 0), cap);
        const int q_max = a.q_stride > 0 ? a.q_stride : a.n_tokens;
        if (q < 0 || q > q_max) bad = true, q = min(max(q, 0), q_max);
        if (a.q_stride > 0 && q > 0 && b * a.q_stride + q > a.n_tokens) bad = true;
        const int need = (kv + a.page_size - 1) / a.page_size, held = a.held[b], had = min(max(held, 0), a.table_ld);
        if (held != had) bad = true;
        const int v[3] = {max(had - need, 0), max(need - had, 0), q};
        back[b] = v[0], want[b] = v[1], toks[b] = v[2];
        base[b] = min(had, need);
#pragma unroll
        for (int i = 0; i < 3; ++i) s[i] = plan_add(i == 2, s[i], v[i]);
    }
    int incl[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        incl[i] = s[i];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, incl[i], o);
            if (lane >= o) incl[i] = plan_add(i == 2, incl[i], u);
        }
        if (lane == 31) wsum[i][warp] = incl[i];
    }
    __syncthreads();
    int tot[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        int before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < kPlanThreads / 32; ++w) {
            const int u = wsum[i][w];
            before = w < warp ? plan_add(i == 2, before, u) : before;
            all = plan_add(i == 2, all, u);
        }
        tot[i] = all;
        int in_front = incl[i] - s[i];
        if (i == 2) in_front = __shfl_up_sync(0xffffffffu, incl[i], 1);
        int run = plan_add(i == 2, before, i == 2 && lane == 0 ? 0 : in_front);
        int* arr = i == 0 ? back : i == 1 ? want : toks;
        for (int b = b0; b < b1; ++b) {
            const int v = arr[b];
            arr[b] = run;
            run = plan_add(i == 2, run, v);
        }
        if (tid == 0) arr[n] = all;
    }
    __syncthreads();
    const int n_back = tot[0], n_want = tot[1], n_tok = tot[2];
    const int count0 = min(max(free0, 0), a.n_pages), room = a.n_pages - count0;
    const int count = count0 + min(n_back, room), left = max(count - n_want, 0);
    if (free0 != count0 || n_back > room) bad = true;  // also: the stack would hold more pages than there are
    if (n_back | n_want) {
        cluster.sync();  // every CTA has read the old state
        for (unsigned k0 = gtid; k0 < (unsigned)n_back; k0 += 4 * gn) {
            size_t i[4];
            int page[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const unsigned k = k0 + u * gn;
                if (k >= (unsigned)n_back) continue;
                const int b = owner(back, n, (int)k);
                i[u] = (size_t)b * a.table_ld + base[b] + ((int)k - back[b]);
                page[u] = a.table[i[u]];
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const unsigned k = k0 + u * gn;
                if (k >= (unsigned)n_back) continue;
                if (k < (unsigned)room) a.free_pages[count0 + k] = page[u];
                a.table[i[u]] = -1;
            }
        }
        if (n_back && n_want) cluster.sync();  // what was given back can be taken
        for (int k0 = gtid; k0 < min(n_want, count); k0 += 4 * gn) {
            size_t i[4];
            int page[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int k = k0 + u * gn;
                if (k >= n_want || k >= count) continue;
                page[u] = a.free_pages[count - 1 - k];
                const int b = owner(want, n, k);
                i[u] = (size_t)b * a.table_ld + base[b] + (k - want[b]);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int k = k0 + u * gn;
                if (k >= n_want || k >= count) continue;
                a.table[i[u]] = page[u];
                a.free_pages[count - 1 - k] = -1;
            }
        }
        for (int b = gtid; b < n; b += gn) {
            const int w = want[b + 1] - want[b];
            a.held[b] = base[b] + min(max(count - want[b], 0), w);
        }
        if (gtid == 0) *a.n_free = left;
        cluster.sync();  // the new table
    }
    if (gtid == 0) {
        if (a.missing) *a.missing = max(n_want - count, 0);
        if (a.q_stride == 0 && n_tok > a.n_tokens) bad = true;
    }
    for (int b = gtid; b < n; b += gn) a.q_start[b] = a.q_stride > 0 ? b * a.q_stride : toks[b];
    for (unsigned u = gtid; u < (unsigned)a.n_tokens; u += gn) {
        const int k = (int)u;
        int b, t;
        bool live;
        if (a.q_stride > 0) {
            b = k / a.q_stride;
            t = k - b * a.q_stride;
            live = b < n;
        } else {
            b = owner(toks, n, k);
            t = k - toks[b];
            live = true;
        }
        int slot = -1, pos = -1;
        int q = live ? toks[b + 1] - toks[b] : 0;
        if (live && toks[b + 1] == INT32_MAX) q = min(max(a.q_len[b], 0), a.q_stride > 0 ? a.q_stride : a.n_tokens);
        if (t >= 0 && t < q) {
            const int p = min(a.kv_len[b], cap) - q + t;
            if (p >= 0 && p < cap) {
                pos = a.pos0 + p;
                const int page = a.table[(size_t)b * a.table_ld + p / a.page_size];
                if (page >= 0 && page < a.n_pages) slot = page * a.page_size + p % a.page_size;
                else if (page != -1) bad = true;
            }
        }
        a.slots[k] = slot;
        if (a.positions) a.positions[k] = pos;
    }
    if (bad) set_dev_error(a.err, DEV_ERR_BAD_ARG);
}

__global__ void k_pages_reset(sd_pages p) {
    const size_t n_tab = (size_t)p.n_req * p.table_ld, step = (size_t)gridDim.x * blockDim.x;
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n_tab; i += step) p.table[i] = -1;
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < (size_t)p.n_pages; i += step)
        p.free_pages[i] = p.n_pages - 1 - (int)i;
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < (size_t)p.n_req; i += step) p.held[i] = 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.n_free = p.n_pages;
}

// ---------------------------------------------------------------------------------------------
// K/V append: a cast copy, bound by HBM (source read once, pool rows written once).  One warp per token, so its slot is
// read once; where pointers and strides allow it, lanes move 8 elements at a time and the row's loads are all in flight
// before the first store.  16384 tokens of 2 x 1024 bf16: 24.6 us, 5.5 TB/s (110 us with one element per lane).
// ---------------------------------------------------------------------------------------------
struct AppendArgs {
    const void *k, *v;
    void *kp, *vp;
    int64_t k_ld, v_ld, page_stride, pos_stride, head_stride;
    int n_kv, hd, page_size, n_slots, n_tokens;
    const int32_t* slots;
    int* err;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Eight elements as the pool's type.
template <class S, class T>
struct Eight {
    uint4 v;
    __device__ __forceinline__ void load(const S* p) {
        if constexpr (sizeof(S) == 2) {
            v = __ldg(reinterpret_cast<const uint4*>(p));
        } else {
            const float4 x = __ldg(reinterpret_cast<const float4*>(p)), y = __ldg(reinterpret_cast<const float4*>(p) + 1);
            T t[8] = {from_f32<T>(x.x), from_f32<T>(x.y), from_f32<T>(x.z), from_f32<T>(x.w),
                      from_f32<T>(y.x), from_f32<T>(y.y), from_f32<T>(y.z), from_f32<T>(y.w)};
            v = *reinterpret_cast<const uint4*>(t);
        }
    }
};

// VEC: 8 elements per lane (16-byte aligned rows and heads); else one.
template <class S, class T, bool VEC>
__global__ void __launch_bounds__(256) k_kv_append(const AppendArgs a) {
    const int lane = threadIdx.x & 31;
    const long long tok = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    if (tok >= a.n_tokens) return;
    const int slot = a.slots[tok];
    if (slot < 0 || slot >= a.n_slots) {
        if (slot != -1 && lane == 0) set_dev_error(a.err, DEV_ERR_BAD_ARG);
        return;
    }
    const size_t dst = (size_t)(slot / a.page_size) * a.page_stride + (size_t)(slot % a.page_size) * a.pos_stride;
    const bool dense = a.head_stride == a.hd;
    auto at = [&](int e) {  // element e of a row in the pool
        if (dense) return dst + e;
        const int h = e / a.hd;
        return dst + (size_t)h * a.head_stride + (e - h * a.hd);
    };
    const S *k = static_cast<const S*>(a.k) + (size_t)tok * a.k_ld, *v = static_cast<const S*>(a.v) + (size_t)tok * a.v_ld;
    T *kp = static_cast<T*>(a.kp), *vp = static_cast<T*>(a.vp);
    const int row = a.n_kv * a.hd;
    if constexpr (VEC) {
        constexpr int U = 4;
        for (int e0 = lane * 8; e0 < row; e0 += 32 * 8 * U) {
            Eight<S, T> x[2][U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (e0 + u * 256 < row) {
                    x[0][u].load(k + e0 + u * 256);
                    x[1][u].load(v + e0 + u * 256);
                }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (e0 + u * 256 < row) {
                    const size_t d = at(e0 + u * 256);
                    *reinterpret_cast<uint4*>(kp + d) = x[0][u].v;
                    *reinterpret_cast<uint4*>(vp + d) = x[1][u].v;
                }
        }
    } else {
        for (int e = lane; e < row; e += 32) {
            const size_t d = at(e);
            kp[d] = from_f32<T>(to_f32(k[e]));
            vp[d] = from_f32<T>(to_f32(v[e]));
        }
    }
}

template <class S, class T>
void launch_append(const AppendArgs& a, bool vec, cudaStream_t st) {
    const int grid = (a.n_tokens + 7) / 8;
    if (vec) k_kv_append<S, T, true><<<grid, 256, 0, st>>>(a);
    else k_kv_append<S, T, false><<<grid, 256, 0, st>>>(a);
}

}  // namespace

int launch_pages_plan(const sd_pages* p, const int32_t* kv_len, const int32_t* q_len, int q_stride, int pos0, int n_tokens,
                      int32_t* q_start, int32_t* slots, int32_t* positions, int32_t* missing, int* err, cudaStream_t st) {
    PlanArgs a{p->table, p->held, p->free_pages, p->n_free, p->n_req, p->table_ld, p->n_pages, p->page_size,
               kv_len, q_len, q_stride, pos0, n_tokens, q_start, slots, positions, missing, err};
    const size_t smem = plan_smem(p->n_req);
    cudaError_t e = cudaSuccess;
    if (smem > 48 * 1024 - 1024) {
        // once per device, to the largest batch's: another thread's smaller batch must not lower it in front of a launch
        static std::atomic<bool> ready[64];
        int dev = 0;
        if ((e = cudaGetDevice(&dev)) != cudaSuccess) return cuda_fail(e, "pages plan");
        if (dev < 0 || dev >= 64 || !ready[dev].load(std::memory_order_acquire)) {
            e = cudaFuncSetAttribute(k_pages_plan, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)plan_smem(SD_PAGES_MAX_REQ));
            if (e != cudaSuccess) return cuda_fail(e, "pages plan");
            if (dev >= 0 && dev < 64) ready[dev].store(true, std::memory_order_release);
        }
    }
    // a thread's share of a step is a token or a few pages of a request (the host does not know how many move)
    const long long items = std::max<long long>(n_tokens, 16LL * p->n_req);
    int ctas = 1;
    while (ctas < 8 && ctas * kPlanThreads < items) ctas *= 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kPlanThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = ctas;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, k_pages_plan, (const PlanArgs)a);
    return e == cudaSuccess ? SD_OK : cuda_fail(e, "pages plan");
}

}  // namespace sd

extern "C" {

int sd_pages_reset_dev(const sd_pages* p, void* stream) {
    clear_error();
    int rc = check_pages(p, "sd_pages_reset_dev"), dev;
    if (rc || (rc = paged_device(p->table, "sd_pages_reset_dev", &dev))) return rc;
    k_pages_reset<<<device_sm_count(dev), 256, 0, (cudaStream_t)stream>>>(*p);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? SD_OK : cuda_fail(e, "pages reset");
}

int sd_pages_plan_dev(const sd_pages* p, const int32_t* kv_len, const int32_t* q_len, int q_stride, int pos0, int n_tokens,
                      int32_t* q_start, int32_t* slots, int32_t* positions, int32_t* missing, void* stream) {
    clear_error();
    int rc = check_pages(p, "sd_pages_plan_dev"), dev;
    if (rc) return rc;
    if (!kv_len || !q_len || !q_start || n_tokens < 0 || (n_tokens > 0 && !slots) || q_stride < 0 || pos0 < 0)
        return fail(SD_ERR_INVALID, "sd_pages_plan_dev: bad arguments");
    if ((int64_t)p->n_req * q_stride > INT32_MAX || (int64_t)pos0 + (int64_t)p->table_ld * p->page_size > INT32_MAX)
        return fail(SD_ERR_INVALID, "sd_pages_plan_dev: q_stride %d or pos0 %d too large", q_stride, pos0);
    if ((rc = paged_device(p->table, "sd_pages_plan_dev", &dev))) return rc;
    return launch_pages_plan(p, kv_len, q_len, q_stride, pos0, n_tokens, q_start, slots, positions, missing, device_error_word(dev),
                             (cudaStream_t)stream);
}

int sd_kv_append_dev(const sd_kv_pool* pool, const void* k, const void* v, int src_dtype, int64_t k_ld, int64_t v_ld,
                     const int32_t* slots, int n_tokens, void* stream) {
    clear_error();
    int rc = check_kv_pool(pool, "sd_kv_append_dev"), dev;
    if (rc) return rc;
    if (n_tokens < 0 || (n_tokens > 0 && (!k || !v || !slots))) return fail(SD_ERR_INVALID, "sd_kv_append_dev: bad arguments");
    if (src_dtype != SD_F32 && src_dtype != pool->dtype)
        return fail(SD_ERR_INVALID, "sd_kv_append_dev: source type %d for a pool of type %d", src_dtype, pool->dtype);
    if (n_tokens == 0) return SD_OK;
    if ((rc = paged_device(pool->k, "sd_kv_append_dev", &dev))) return rc;
    AppendArgs a{k, v, pool->k, pool->v, k_ld, v_ld, pool->page_stride, pool->pos_stride, pool->head_stride,
                 pool->n_kv_heads, pool->head_dim, pool->page_size, pool->n_pages * pool->page_size, n_tokens, slots,
                 device_error_word(dev)};
    const cudaStream_t st = (cudaStream_t)stream;
    const int per16 = src_dtype == SD_F32 ? 4 : 8;  // source elements in 16 bytes
    auto al = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
    const bool vec = al(k) && al(v) && al(pool->k) && al(pool->v) && k_ld % per16 == 0 && v_ld % per16 == 0 &&
                     pool->page_stride % 8 == 0 && pool->pos_stride % 8 == 0 && pool->head_stride % 8 == 0;
    if (pool->dtype == SD_F16) {
        if (src_dtype == SD_F32) launch_append<float, __half>(a, vec, st);
        else launch_append<__half, __half>(a, vec, st);
    } else {
        if (src_dtype == SD_F32) launch_append<float, __nv_bfloat16>(a, vec, st);
        else launch_append<__nv_bfloat16, __nv_bfloat16>(a, vec, st);
    }
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? SD_OK : cuda_fail(e, "kv append");
}

}  // extern "C"
