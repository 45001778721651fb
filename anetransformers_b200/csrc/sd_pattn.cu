// sd_pattn.cu -- attention over a paged K/V cache: grouped heads, a prefix shared by every request of the batch,
// tanh-capped and distance-biased scores, windows.
//
//   o_t = sum_j p_j v_j / sum_j p_j,  p_j = exp(z_j - max z),
//   z_j = f(scale q_t.k_j) - slope (pos_t - pos_j),  f(s) = cap tanh(s / cap) or s
// over the visible j: prefix positions, then the request's own positions up to the row's, less those at a distance
// of `window` or more.
#include <cuda.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
#include <type_traits>

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

// ---------------------------------------------------------------------------------------------
// Tensor-core kernel (head_dim 64 and 128): tcgen05.mma with S, P and O in tensor memory, K/V tiles by TMA.
//
// Rows.  The query rows of one kv head are (token, head of its group); a tile holds TPT = 128 / G tokens, TPT * G
// rows of the MMA's M = 128.  Keys come in tiles of 128.  Work items:
//   own items      (request, row tiles, kv head, chunk of its keys)
//   prefix items   (row tiles over the whole step's tokens, kv head, chunk of the prefix): the shared prefix is read
//                  once for the rows of all requests.  A request with more rows than two tiles fills them by itself
//                  and takes the prefix tiles in front of its own ("inline", one softmax over both).
// An item of more than TPT tokens is a pair: slot 0 and 1 (accumulators and softmax warpgroups) take a row tile
// each and share every K/V tile.  A smaller one has one row tile: slot 0 takes its even key tiles, slot 1 the odd
// ones, and slot 0 merges the two states at the end.  Rows whose keys lie in several items leave (max, sum, O) in
// the workspace for k_pattn_combine; others are written by their item.
//
// Warps (12): 0-3 softmax of slot 0, 4-7 of slot 1 (thread = row), 8 TMA and the handing out of items, 9 and 11 MMA
// issue of slot 0 and 1, 10 zeroes V rows that no row may see (0 x NaN is NaN in the product).  P overwrites S in
// tensor memory and is the A operand of P V.
// The running maximum that O refers to moves only when a row's maximum rises by more than 2^8 (exact: O and the sum
// refer to the same value), so O is rarely rescaled.  Every wait is bounded in time (sd_common.cuh).
//
// What bounds it.  One causal prompt of 9472 tokens, 32 / 8 heads of 128, no bias: 636 us, 1154 TFLOP/s in short bursts (0.70
// of the measured burst rate of a matrix product); back to back under the power limit 734 us, 0.72 of the sustained one.
// 256 rows x 128 keys take the tensor cores 2480 clk with S in halves of 64 keys (N = 64, bound by shared memory; 2050 in one
// piece) and the exponentials 2048 clk; each softmax warp needs about 1900 clk per half, of them 500 to 1000 waiting for
// its share of the exponentials.  With caps and biases the extra arithmetic per score bounds it.
//
// What the steps measured, each against the kernel as it was then.  S in halves: prompts gained, since a slot's softmax
// then overlaps its own MMAs (588 -> 550, capped 356 -> 302, biased 476 -> 441 us); single tokens lost (32 over one prefix
// of 32768 keys 89 -> 97 us, 64 over ragged contexts 410 -> 547 us), and k_pattn_rows serves all but their shared prefix now.
// With S in halves, part of the exponentials on the FMA pipe (every third to eighth pair): biased 2 % faster, the others unchanged to 5 % slower, capped
// 5 to 10 % slower; not kept.  16 softmax warps of half a row each: 570 -> 695 us; not kept.
// ---------------------------------------------------------------------------------------------
constexpr int kPaThreads = 384;
constexpr int kPaKeys = 128;        // keys per tile
constexpr int kPaHalf = 128 * 128;  // bytes of 128 rows x 64 elements (one 128-byte swizzle row each)

struct PaArgs {
    CUtensorMap tq, tk, tv;
    sd_attn_args a;
    int G, TPT;            // query heads per kv head, tokens per row tile
    int np;                // key tiles of the prefix
    int n_pt, cp, ct_pre;  // prefix items: row-tile pairs over the tokens, chunks, tiles per chunk
    int ct_own;            // tiles per chunk of own items
    bool few;              // own items by k_pattn_rows
    // States of rows whose keys lie in several items, by split; row (kv head, token, head of its group), so that the rows
    // of a tile, one per thread, are neighbours: O as float4 [splits][hd / 4][rows], (max, sum) as [splits][rows].
    float4* acc;
    float2* ml;
    int* err;
};

struct alignas(16) PaItem {
    int b, kvh, tok0, ntok;   // request (-1: prefix item), kv head, first token, tokens
    int pair, direct;
    int v0, n, npt;           // first key tile, their number; tiles below npt are the prefix's
    int klo_p, klo_o, khi_o;  // keys outside [klo_p, prefix_len) and [klo_o, khi_o) are seen by no row of the item
    int base;                 // kv - q: own position of the request's first row
    int q0, rows;             // the request's first token and its tokens
    int split;
};

struct PaCtl {
    uint64_t qfull[2], qempty[2];  // per Q tile buffer
    uint64_t full[16], empty[16], fixed[16];
    uint64_t sfull[2][2], pready[2][2];  // [slot][half of the tile's keys]: S and P written
    // A parity wait tells a phase from its neighbour only: ofull (one phase per half's product) is waited for where the
    // last but one product is known to be complete, odone has one phase per item.
    uint64_t ofull[2], odone[2];
    uint64_t mready, mdone, done;
    uint64_t ifull, iempty, claim;  // hand-over of the next item; answer to the claim of another CTA's
    uint4 claimed;
    PaItem item;  // ntok 0: no more
    // per key tile (in turn) and half: which of its 16-key groups were loaded (bits 0-3), and whether V has rows that no
    // row of the item may see (bit 8)
    uint32_t okmask[16][2];
    int pages[16][8];   // per key tile: its page ids, -1 where there is none to load
    uint64_t fq[16];    // a request for zero rows is posted
    int4 fix[16];       // stage (-1: no more), its phase, first and last + 1 row to keep | mask << 16
    float2 ml1[128];      // slot 1's state at a merge
    uint32_t tmem;
    int abort;
    int wsum[16];
};

__device__ __forceinline__ int pa_q(const sd_attn_args& a, int b) { return min(max(a.q_len[b], 0), a.max_q); }
__device__ __forceinline__ int pa_kv(const sd_attn_args& a, int b) { return min(max(a.kv_len[b], 0), a.max_kv); }
__device__ __forceinline__ int pa_rows(const sd_attn_args& a, int b) {
    return max(0, min(pa_q(a, b), a.n_tokens - max(a.q_start[b], 0)));
}
__device__ __forceinline__ bool pa_inline(const PaArgs& p, int rows) { return p.a.prefix_len > 0 && rows > 2 * p.TPT; }
__device__ __forceinline__ int pa_tiles(const PaArgs& p, int rows) {
    return rows <= p.TPT ? (rows > 0) : (rows + 2 * p.TPT - 1) / (2 * p.TPT);
}
// Chunks of a request's key tiles (the prefix's in front if it is inline) and tiles per chunk: as equal as they can be,
// but with a window on a fixed grid, of which each item sees a part.
__device__ __forceinline__ int pa_chunks(const PaArgs& p, int kv, bool inl, int* size) {
    const int t = (kv + kPaKeys - 1) / kPaKeys + (inl ? p.np : 0);
    const int n = max(1, (t + p.ct_own - 1) / p.ct_own);
    *size = p.a.window > 0 || p.few ? p.ct_own : (t + n - 1) / n;
    return n;
}
__device__ __forceinline__ int pa_request(const sd_attn_args& a, int tok) {
    int lo = 0, hi = a.n_req;
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (a.q_start[m] <= tok) lo = m; else hi = m;
    }
    return lo;
}

// First prefix position that a row of a prefix item sees through the window: from the least position of its rows that have
// one, but for inline requests', whose prefix is in their own items.  A whole warp does this, a request per lane.  (A call
// of its own: inlined, it cost calls without a window 2 to 3 % by the code around it.)
__device__ __noinline__ int pa_prefix_first(const PaArgs& p, int tok0, int ntok, int lane) {
    const sd_attn_args& a = p.a;
    int first = 0, last = a.n_req - 1, low = INT32_MAX;
    if (a.n_req > 256) {  // two lanes search at once; fewer requests are looked at without a search (its loads follow one another)
        const int edge = pa_request(a, lane & 1 ? tok0 + ntok - 1 : tok0);
        first = __shfl_sync(0xffffffffu, edge, 0);
        last = __shfl_sync(0xffffffffu, edge, 1);
    }
#pragma unroll 2
    for (int b = first + lane; b <= last; b += 32) {
        const int start = a.q_start[b], rows = pa_rows(a, b), base = pa_kv(a, b) - pa_q(a, b);
        const int t0 = max(0, tok0 - start), t1 = min(rows, tok0 + ntok - start);
        if (t0 < t1 && base + t1 > 0 && !pa_inline(p, rows)) low = min(low, max(0, base + t0));
    }
    low = __reduce_min_sync(0xffffffffu, low);
    return low == INT32_MAX ? a.prefix_len : min(a.prefix_len, max(0, a.prefix_len + low + 1 - a.window));
}

// Item number i of the launch; false if it holds nothing (prefix rows of an inline request).  The TMA warp does this, ahead
// of the others; they read the result.
__device__ __forceinline__ bool pa_item(const PaArgs& p, const int* ustart, int i, int lane, PaItem& it) {
    const sd_attn_args& a = p.a;
    const int n_kv = a.pool.n_kv_heads, P = a.prefix_len, W = a.window;
    const int n_pre = p.cp * p.n_pt * n_kv;
    if (i < n_pre) {
        it.kvh = i % n_kv;
        const int u = i / n_kv, c = u / p.n_pt;
        it.tok0 = (u - c * p.n_pt) * 2 * p.TPT;
        it.ntok = min(2 * p.TPT, a.n_tokens - it.tok0);
        if (a.max_q > 2 * p.TPT) {
            const int b = pa_request(a, it.tok0), rows = pa_rows(a, b);
            if (pa_inline(p, rows) && it.tok0 >= a.q_start[b] && it.tok0 + it.ntok <= a.q_start[b] + rows) return false;
        }
        it.b = -1;
        it.pair = it.ntok > p.TPT;
        it.direct = false;
        it.npt = p.np;
        it.klo_p = W > 0 ? pa_prefix_first(p, it.tok0, it.ntok, lane) : 0;
        it.klo_o = it.khi_o = 0;
        it.v0 = max(c * p.ct_pre, it.klo_p / kPaKeys);
        it.n = max(0, min(p.np, (c + 1) * p.ct_pre) - it.v0);
        if (it.klo_p >= P) it.n = 0;
        it.base = it.q0 = it.rows = 0;
        it.split = c;
        return true;
    }
    i -= n_pre;
    it.kvh = i % n_kv;
    const int u = i / n_kv;
    int lo = 0, hi = a.n_req;
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (ustart[m] <= u) lo = m; else hi = m;
    }
    const int b = lo, local = u - ustart[b];
    const int q = pa_q(a, b), kv = pa_kv(a, b), rows = pa_rows(a, b), nt = pa_tiles(p, rows);
    const bool inl = pa_inline(p, rows);
    const int c = local / nt, tile = nt - 1 - (local - c * nt);  // the tiles with most keys first
    int size;
    const int chunks = pa_chunks(p, kv, inl, &size);
    it.b = b;
    it.q0 = max(a.q_start[b], 0);
    it.rows = rows;
    it.base = kv - q;
    it.tok0 = it.q0 + tile * 2 * p.TPT;
    it.ntok = min(2 * p.TPT, rows - tile * 2 * p.TPT);
    it.pair = it.ntok > p.TPT;
    it.direct = chunks == 1 && (P == 0 || inl);
    it.npt = inl ? p.np : 0;
    const int last = it.base + tile * 2 * p.TPT + it.ntok - 1;
    const int first = max(0, it.base + tile * 2 * p.TPT);  // of the rows that have a position
    it.khi_o = max(0, last + 1);
    it.klo_o = W > 0 ? max(0, first + 1 - W) : 0;
    it.klo_p = W > 0 ? min(P, max(0, P + first + 1 - W)) : 0;
    int s0 = it.klo_o / kPaKeys + it.npt;
    if (inl && it.klo_p < P) s0 = it.klo_p / kPaKeys;
    it.v0 = max(c * size, s0);
    const int end = min((c + 1) * size, it.npt + (it.khi_o + kPaKeys - 1) / kPaKeys);
    it.n = last < 0 ? 0 : max(0, end - it.v0);
    it.split = p.cp + c;
    return true;
}

// Keys [k0, k0 + 128) of the item's t-th tile, and which of them its rows may see.  The nearest keys come first: with a
// distance bias the largest scores then do too, and O keeps its scale (measured at the 2 x 2048-token biased prompts).
struct PaTile {
    bool prefix;
    int k0, lo, hi;
};
__device__ __forceinline__ PaTile pa_tile(const PaArgs& p, const PaItem& it, int t) {
    const int v = it.v0 + it.n - 1 - t;
    PaTile k;
    k.prefix = v < it.npt;
    k.k0 = (k.prefix ? v : v - it.npt) * kPaKeys;
    k.lo = k.prefix ? it.klo_p : it.klo_o;
    k.hi = k.prefix ? p.a.prefix_len : it.khi_o;
    return k;
}

// Waits of one thread and of a whole warp; false once any wait of the CTA has run out.
__device__ __noinline__ bool pa_wait_slow(uint64_t* bar, uint32_t parity, PaCtl* ctl, int* err, int code) {
    if (*(volatile int*)&ctl->abort) return false;
    if (mbar_wait(bar, parity)) return true;
    set_dev_error(err, code);
    *(volatile int*)&ctl->abort = 1;
    return false;
}
__device__ __forceinline__ bool pa_wait(uint64_t* bar, uint32_t parity, PaCtl* ctl, int* err, int code) {
    return mbar_try_wait(bar, parity) || pa_wait_slow(bar, parity, ctl, err, code);
}
__device__ __forceinline__ bool pa_wait_warp(uint64_t* bar, uint32_t parity, PaCtl* ctl, int* err, int code) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    return __all_sync(0xffffffffu, pa_wait_slow(bar, parity, ctl, err, code));
}

// The CTA's k-th item, for a warp and for one thread; false after the last (or when a wait ran out).  Ten take each item;
// with the last of them the TMA warp may hand out the next one.
__device__ __forceinline__ bool pa_next(PaCtl* ctl, int k, int lane, int* err, PaItem& it) {
    if (!pa_wait_warp(&ctl->ifull, k & 1, ctl, err, DEV_ERR_FULL_WAIT)) return false;
    it = ctl->item;
    __syncwarp();
    if (lane == 0) mbar_arrive(&ctl->iempty);
    return it.ntok > 0;
}
__device__ __forceinline__ bool pa_next_thread(PaCtl* ctl, int k, int* err, PaItem& it) {
    if (!pa_wait(&ctl->ifull, k & 1, ctl, err, DEV_ERR_FULL_WAIT)) return false;
    it = ctl->item;
    mbar_arrive(&ctl->iempty);
    return it.ntok > 0;
}
// Claim a CTA of the grid that has not started (cluster launch control); the answer lands in ctl->claimed.
__device__ __forceinline__ void pa_claim(PaCtl* ctl) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    mbar_arrive_expect_tx(&ctl->claim, 16);
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                     smem_u32(&ctl->claimed)),
                 "r"(smem_u32(&ctl->claim))
                 : "memory");
}
__device__ __forceinline__ int pa_claimed(PaCtl* ctl) {  // its index, or -1 if there is none left
    uint32_t got, x;
    asm volatile(
        "{\n .reg .pred p;\n .reg .b128 r;\n ld.shared.b128 r, [%2];\n"
        " clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n selp.u32 %0, 1, 0, p;\n"
        " mov.u32 %1, 0;\n @p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n}\n"
        : "=r"(got), "=r"(x)
        : "r"(smem_u32(&ctl->claimed))
        : "memory");
    return got ? (int)x : -1;
}

__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* m, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(m), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
        : "memory");
}
__device__ __forceinline__ void tma_5d(uint32_t dst, const CUtensorMap* m, int x, int y, int z, int w, int v, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(
            dst),
        "l"(m), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v)
        : "memory");
}

// Shared-memory matrix descriptor of a 128-byte swizzled operand (rows of 64 16-bit elements): start address, leading
// and stride byte offsets in 16-byte units, bit 46 the descriptor version of sm_100, bits 61-63 the swizzle.
// K-major (Q, K): stride = 1024 between groups of 8 rows.  MN-major (V, read by columns): leading = the distance
// between blocks of 64 columns, stride = 1024 between groups of 8 keys.
// The high word is the same for both; the low word is the start address and the leading offset, so that a step along K
// is one 32-bit add.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t sw128_lo(uint32_t addr, uint32_t lbo) { return (addr >> 4) | ((lbo >> 4) << 16); }
// Instruction descriptor of kind::f16: D fp32, A and B fp16 or bf16, B MN-major if trans_b, M = 128.
__host__ __device__ constexpr uint32_t idesc_f16(bool bf16, int n, bool trans_b) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((trans_b ? 1u : 0u) << 16) |
           ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 da, db;\n setp.ne.b32 p, %4, 0;\n mov.b64 da, {%1, %5};\n mov.b64 db, {%2, %5};\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(kDescHi)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 db;\n setp.ne.b32 p, %4, 0;\n mov.b64 db, {%2, %5};\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(kDescHi)
        : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t e;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(e));
    return e != 0;
}
__device__ __forceinline__ void pa_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void pa_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pa_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pa_ld32(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr));
}
// The loads' registers pass through the wait, so that no use of them moves in front of it.
__device__ __forceinline__ void pa_wait_ld(uint32_t (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                   "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]),
                   "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]),
                   "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]),
                   "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void pa_st32(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
        "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(v[0]),
        "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
        "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]),
        "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]),
        "r"(v[29]), "r"(v[30]), "r"(v[31]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void pa_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// cap tanh(x) of two values with |x| <= 1/2: x times a polynomial in x^2 (minimax, relative error 6.4e-7) times the cap.
struct CapPoly {
    float2 c0, c1, c2, c3;
};
__device__ __forceinline__ CapPoly cap_poly(float cap) {
    const float a = -0.33328160643577576f * cap, b = 0.13205359876155853f * cap, c = -0.0447506457567215f * cap;
    return CapPoly{make_float2(cap, cap), make_float2(a, a), make_float2(b, b), make_float2(c, c)};
}
__device__ __forceinline__ float2 cap_small(float2 x, const CapPoly& k) {
    const float2 u = __fmul2_rn(x, x);
    float2 q = __ffma2_rn(u, k.c3, k.c2);
    q = __ffma2_rn(u, q, k.c1);
    q = __ffma2_rn(u, q, k.c0);
    return __fmul2_rn(x, q);
}
template <class T> __device__ __forceinline__ uint32_t pa_pack(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pa_pack<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pa_pack<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <int HD>
constexpr int pa_stages() { return HD == 128 ? 8 : 16; }
template <int HD>
constexpr size_t pa_smem(int n_req) {
    return (size_t)2 * (HD / 64) * kPaHalf + (size_t)pa_stages<HD>() * (HD / 64) * (kPaHalf / 2) + sizeof(PaCtl) +
           ((size_t)n_req + 1) * 4 + 1024;
}

// MOD: capped or biased scores, or a scale that is not positive (then the maximum is not that of q.k).
template <class T, int HD, bool MOD>
__global__ void __launch_bounds__(kPaThreads, 1) k_pattn(const __grid_constant__ PaArgs p) {
    constexpr int NST = pa_stages<HD>();
    constexpr int NH = HD / 64;                 // 64-element halves of a row
    constexpr uint32_t TILE = NH * kPaHalf;     // bytes of a Q tile
    constexpr uint32_t STAGE = TILE / 2;        // bytes of a ring stage: K or V of 64 keys, [64-element half][key]
    constexpr uint32_t kSHalf = kPaHalf / 2;
    constexpr bool BF = sizeof(T) == 2 && !std::is_same<T, __half>::value;
    // fp16 weights are kept 2^6 above the running maximum's scale (at most 2^14 with the 2^8 slack), so that small
    // ones stay in the type's normal range
    constexpr float kShift = BF ? 0.f : 6.f;
    constexpr float kSlack = 8.f;
    extern __shared__ uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t qs = smem_u32(smem), kvs = qs + 2 * TILE;
    PaCtl* ctl = reinterpret_cast<PaCtl*>(smem + 2 * TILE + NST * STAGE);
    int* ustart = reinterpret_cast<int*>(ctl + 1);
    const sd_attn_args& a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&ctl->qfull[i], 1);
            mbar_init(&ctl->qempty[i], 2);
        }
        for (int i = 0; i < NST; ++i) {
            mbar_init(&ctl->full[i], 1);
            mbar_init(&ctl->empty[i], 2);
            mbar_init(&ctl->fixed[i], 1);
        }
        for (int i = 0; i < 16; ++i) mbar_init(&ctl->fq[i], 1);
        for (int i = 0; i < 2; ++i) {
            for (int h = 0; h < 2; ++h) {
                mbar_init(&ctl->sfull[i][h], 1);
                mbar_init(&ctl->pready[i][h], 4);
            }
            mbar_init(&ctl->ofull[i], 1);
            mbar_init(&ctl->odone[i], 1);
        }
        mbar_init(&ctl->mready, 128);
        mbar_init(&ctl->mdone, 128);
        mbar_init(&ctl->done, 2);
        mbar_init(&ctl->ifull, 1);
        mbar_init(&ctl->iempty, 10);
        mbar_init(&ctl->claim, 1);
        ctl->abort = 0;
        fence_mbar_init();
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&ctl->tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // units (row tiles x chunks) of each request: exclusive sums
    {
        const int n = a.n_req, per = (n + kPaThreads - 1) / kPaThreads;
        const int b0 = min(n, tid * per), b1 = min(n, b0 + per);
        int sum = 0;
        bool bad = false;
        for (int b = b0; b < b1; ++b) {
            int size;
            const int rows = p.few ? 0 : pa_rows(a, b);
            const int u = rows > 0 ? pa_tiles(p, rows) * pa_chunks(p, pa_kv(a, b), pa_inline(p, rows), &size) : 0;
            bad |= !p.few && (a.q_len[b] > a.max_q || a.q_len[b] < 0 || a.kv_len[b] > a.max_kv || a.kv_len[b] < 0 ||
                              a.q_start[b] < 0 || rows < pa_q(a, b));
            ustart[b] = u;
            sum += u;
        }
        if (bad && blockIdx.x == 0) set_dev_error(p.err, DEV_ERR_BAD_ARG);
        int incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) ctl->wsum[warp] = incl;
        __syncthreads();
        int before = 0;
        for (int w = 0; w < warp; ++w) before += ctl->wsum[w];
        int run = before + incl - sum;
        for (int b = b0; b < b1; ++b) {
            const int u = ustart[b];
            ustart[b] = run;
            run += u;
        }
        if (tid == kPaThreads - 1) ustart[n] = before + incl;
    }
    pa_fence_before();
    __syncthreads();
    pa_fence_after();
    pdl_trigger();
    const uint32_t tmem = ctl->tmem;
    const int n_items = (p.cp * p.n_pt + ustart[a.n_req]) * a.pool.n_kv_heads;
    const int ps = a.pool.page_size, G = p.G;

    if (warp == 8) {
        // ---------------- TMA ----------------
        // One TMA box has at most 64 rows of one page and 128-byte swizzle rows, so 64 elements; it takes the copy engine
        // about 3.1 clk a row and 51 clk a box (measured from L2), so few boxes: both 64-element halves of V rows come in one
        // ([page][half][row], which the product's descriptor can follow page by page), of K rows where a page fills a stage.
        uint32_t pos = 0, tiles = 0, fixes = 0, nq[2] = {0, 0}, qb = 0;
        const int lps = 31 - __clz(ps), box = min(ps, kPaKeys / 2), nb = kPaKeys / 2 / box;  // boxes per stage along the rows
        const int npg = kPaKeys / min(ps, kPaKeys);                                          // pages per tile
        const int nhk = nb == 1 ? 1 : NH;                                                    // boxes of K along the row
        const uint32_t page_bytes = (uint32_t)box * 128u * NH;
        // lane nhk g + j brings part j of the K rows of box g of a stage, lane g the V rows; lane g < npg reads the id of
        // page g of a tile
        const int gk = lane / nhk, jk = lane % nhk;
        const uint32_t dst_k = kvs + jk * kSHalf + gk * box * 128, dst_v = kvs + lane * page_bytes;
        bool ok = true;
        // The grid has one CTA per item; a running CTA takes over CTAs that have not started, so unequal items even out
        // over the SMs and set-up is paid once per SM.
        int next = blockIdx.x < n_items ? (int)blockIdx.x : -1, claims = 0;
        bool open = false;  // a claim is under way
        auto claimed = [&]() {  // the next item's number
            do {
                if (!open && lane == 0) pa_claim(ctl);
                open = true;
                ok = pa_wait_warp(&ctl->claim, claims & 1, ctl, p.err, DEV_ERR_FULL_WAIT);
                if (!ok) return;
                open = false;
                ++claims;
                next = __shfl_sync(0xffffffffu, pa_claimed(ctl), 0);
            } while (next >= n_items);
        };
        for (int k = 0; ok;) {
            PaItem it;
            it.ntok = 0;
            if (next >= 0) {
                if (lane == 0) pa_claim(ctl);
                open = true;
                if (!pa_item(p, ustart, next, lane, it)) {
                    claimed();
                    continue;
                }
            }
            if (lane == 0) {
                ok = k == 0 || pa_wait(&ctl->iempty, (k - 1) & 1, ctl, p.err, DEV_ERR_EMPTY_WAIT);
                if (ok) {
                    ctl->item = it;
                    mbar_arrive(&ctl->ifull);
                }
            }
            ++k;
            ok = __shfl_sync(0xffffffffu, ok, 0);
            if (!ok || it.ntok == 0) break;
            if (it.n == 0) {
                claimed();
                continue;
            }
            const int* own_table = a.table + (size_t)max(it.b, 0) * a.table_ld;
            auto load_ids = [&](int t) {
                if (t >= it.n || lane >= npg) return -2;
                const PaTile kt = pa_tile(p, it, t);
                const int key = kt.k0 + (lane << min(lps, 7));
                if (key >= kt.hi || key + min(ps, kPaKeys) <= kt.lo) return -2;  // nothing of it is seen
                return (kt.prefix ? a.prefix_table : own_table)[key >> lps];
            };
            // the ids of tile t become known to the issuing lanes, its masks to everyone
            auto put_ids = [&](int t, int id) {
                const bool have = id >= 0 && id < a.pool.n_pages;
                if (!have && id != -2) set_dev_error(p.err, DEV_ERR_BAD_ARG);
                if (lane < npg) ctl->pages[(tiles + t) & 15][lane] = have ? id : -1;
                const uint32_t got = __ballot_sync(0xffffffffu, have);
                if (lane < 2) {
                    uint32_t m = 0;  // 16-key groups 4 lane .. 4 lane + 3
#pragma unroll
                    for (int q = 0; q < 4; ++q) m |= (got >> (((4 * lane + q) * 16) >> min(lps, 7)) & 1) << q;
                    const PaTile kt = pa_tile(p, it, t);
                    const int k0 = kt.k0 + lane * 64;
                    ctl->okmask[(tiles + t) & 15][lane] = m | ((k0 < kt.lo || k0 + 64 > kt.hi || m != 0xFu) ? 256u : 0u);
                }
                __syncwarp();
            };
            auto issue = [&](bool v, int t, int h) {
                const int st = pos % NST, g = v ? lane : gk;
                if (pos >= NST && !pa_wait_warp(&ctl->empty[st], (pos / NST - 1) & 1, ctl, p.err, DEV_ERR_EMPTY_WAIT)) {
                    ok = false;
                    return;
                }
                int page = -1, row = 0;
                if (g < nb) {
                    page = ctl->pages[(tiles + t) & 15][lps <= 6 ? h * nb + g : 0];
                    if (lps > 6) row = (pa_tile(p, it, t).k0 & (ps - 1)) + h * 64;
                }
                const uint32_t got = __ballot_sync(0xffffffffu, page >= 0);
                if (lane == 0) {
                    mbar_arrive_expect_tx(&ctl->full[st], __popc(got) * (v || nhk == 1 ? page_bytes : page_bytes / NH));
                    if (v) {
                        const uint32_t m = ctl->okmask[(tiles + t) & 15][h];
                        if (m & 256u) {
                            const PaTile kt = pa_tile(p, it, t);
                            const int k0 = kt.k0 + h * 64;
                            const int l0 = min(max(kt.lo - k0, 0), 64), h0 = min(max(kt.hi - k0, 0), 64);
                            ctl->fix[fixes & 15] = make_int4(st, (pos / NST) & 1, l0, h0 | (int)((m & 0xFu) << 16));
                            mbar_arrive(&ctl->fq[fixes & 15]);
                            ++fixes;
                        }
                    }
                }
                __syncwarp();
                if (page >= 0) tma_5d((v ? dst_v : dst_k) + st * STAGE, v ? &p.tv : &p.tk, 0, row, v ? 0 : jk, it.kvh, page, &ctl->full[st]);
                ++pos;
            };
            const int D = it.pair ? 1 : 2;
            int ids = load_ids(0);
            // Q: both buffers for a pair; single items take turns, so that the next one's Q need not wait for this one
            for (int s = 0; s < 2 && ok; ++s) {
                if (!it.pair && s != (int)qb) continue;
                ok = nq[s] == 0 || pa_wait_warp(&ctl->qempty[s], (nq[s] - 1) & 1, ctl, p.err, DEV_ERR_EMPTY_WAIT);
                if (ok && lane == 0) {
                    mbar_arrive_expect_tx(&ctl->qfull[s], (uint32_t)(NH * p.TPT * G * 128));
                    for (int h = 0; h < NH; ++h)
                        tma_3d(qs + s * TILE + h * kPaHalf, &p.tq, h * 64, it.kvh * G, it.tok0 + (it.pair ? s * p.TPT : 0), &ctl->qfull[s]);
                }
                nq[s] += ok;
            }
            if (!it.pair) qb ^= 1;
            if (!ok) break;
            for (int t = 0; t < D && t < it.n && ok; ++t) {
                put_ids(t, ids);
                ids = load_ids(t + 1);
                issue(false, t, 0);
                if (ok) issue(false, t, 1);
            }
            for (int t = 0; t < it.n && ok; ++t) {
                const int tn = t + D;
                if (tn < it.n) {
                    put_ids(tn, ids);
                    ids = load_ids(tn + 1);  // one tile ahead, so that a stage is refilled as soon as it is free
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    issue(true, t, h);
                    if (ok && tn < it.n) issue(false, tn, h);
                    if (!ok) break;
                }
            }
            tiles += it.n;
            if (ok) claimed();
        }
        if (open) mbar_wait(&ctl->claim, claims & 1);
        if (lane == 0) {  // the zeroing warp may go
            ctl->fix[fixes & 15] = make_int4(-1, 0, 0, 0);
            mbar_arrive(&ctl->fq[fixes & 15]);
        }
        // no copy may still be landing when the CTA exits
        for (uint32_t q = pos > NST ? pos - NST : 0; q < pos; ++q) mbar_wait(&ctl->full[q % NST], (q / NST) & 1);
        for (int s = 0; s < 2; ++s)
            if (nq[s] > 0) mbar_wait(&ctl->qfull[s], (nq[s] - 1) & 1);
    } else if (warp == 9 || warp == 11) {
        // ---------------- MMA issue: one elected thread per slot ----------------
        // A thread's issue of MMAs runs little ahead of the tensor cores, so what it does between them (waits, commits)
        // would leave them idle; with a thread per slot the other's MMAs fill the gaps.
        if (elect_one()) {
            constexpr uint32_t id_s = idesc_f16(BF, kPaKeys / 2, false), id_o = idesc_f16(BF, HD, true);
            const int slot = warp == 9 ? 0 : 1;
            uint32_t pos = 0, fixes = 0, tiles = 0, np = 0, nq[2] = {0, 0}, qb = 0;
            const uint32_t ts = tmem + slot * 128, to = tmem + 256 + slot * HD;
            // 16 keys of V further: within a box [64-element half][row] of up to 64 rows, or in the next page's
            const uint32_t vbox = min(ps, kPaKeys / 2);
            uint32_t vstep[4];
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) vstep[ks] = (ks * 16 / vbox * vbox * 128 * NH + ks * 16 % vbox * 128) >> 4;
            bool ok = true;
            // Both threads walk every stage of the ring, in order, and both release it: a parity wait tells a phase from
            // its neighbour only, so neither may fall a lap behind or get one ahead.
            auto wait_stage = [&]() {
                ok = ok && pa_wait(&ctl->full[pos % NST], (pos / NST) & 1, ctl, p.err, DEV_ERR_FULL_WAIT);
            };
            // S of 64 keys: half h of the slot's next tile, K in the current stage, against Q
            auto score = [&](int h, uint32_t qa) {
                wait_stage();
                if (!ok) return;
                const uint32_t ka = sw128_lo(kvs + (pos % NST) * STAGE, 16);
#pragma unroll
                for (int ks = 0; ks < HD / 16; ++ks)
                    mma_ss(ts + h * 64, qa + (((ks >> 2) * kPaHalf + (ks & 3) * 32) >> 4), ka + (((ks >> 2) * kSHalf + (ks & 3) * 32) >> 4),
                           id_s, ks > 0);
                pa_commit(&ctl->sfull[slot][h]);
                pa_commit(&ctl->empty[pos % NST]);
                ++pos;
            };
            // O += P V over 64 keys (V in the current stage), once V, its unseen rows zero, and P are there
            auto value = [&](int t, int h, bool acc, bool last) {
                wait_stage();
                if (ok && (*(volatile uint32_t*)&ctl->okmask[(tiles + t) & 15][h] & 256u)) {
                    ok = pa_wait(&ctl->fixed[pos % NST], fixes >> (pos % NST) & 1, ctl, p.err, DEV_ERR_FULL_WAIT);
                    fixes ^= 1u << (pos % NST);
                }
                ok = ok && pa_wait(&ctl->pready[slot][h], np & 1, ctl, p.err, DEV_ERR_FULL_WAIT);
                if (!ok) return;
                pa_fence_after();
                const uint32_t va = sw128_lo(kvs + (pos % NST) * STAGE, vbox * 128);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) mma_ts(to, ts + h * 64 + ks * 8, va + vstep[ks], id_o, acc || h > 0 || ks > 0);
                pa_commit(&ctl->ofull[slot]);
                pa_commit(&ctl->empty[pos % NST]);
                if (last && h == 1) pa_commit(&ctl->odone[slot]);
                if (h == 1) ++np;
                ++pos;
            };
            // a stage of the other slot's
            auto pass = [&](bool v, int t, int h) {
                wait_stage();
                if (!ok) return;
                if (v && (*(volatile uint32_t*)&ctl->okmask[(tiles + t) & 15][h] & 256u)) fixes ^= 1u << (pos % NST);
                mbar_arrive(&ctl->empty[pos % NST]);
                ++pos;
            };
            for (int k = 0; ok; ++k) {
                PaItem it;
                if (!pa_next_thread(ctl, k, p.err, it)) break;
                if (it.n == 0) continue;
                // Half tiles of K and V go through the ring in the order of their use: K of the first tile (of the first
                // two of a single item, one per slot), then V of tile t and K of the tile that follows it on its slot,
                // half by half.  Each 64-key half of a slot's tile is an S buffer of its own: its next S follows its
                // product at once, while the softmax is at the other half.
                const int n = it.n, D = it.pair ? 1 : 2, qt = it.pair ? slot : (int)qb;
                // both Q tiles of a pair: a thread that finished ahead of the other must not meet the other's buffer a
                // phase early in the next item
                for (int b = it.pair ? 0 : qt; b <= (it.pair ? 1 : qt); ++b)
                    ok = ok && pa_wait(&ctl->qfull[b], nq[b] & 1, ctl, p.err, DEV_ERR_FULL_WAIT);
                const uint32_t qa = sw128_lo(qs + qt * TILE, 16);
                auto mine = [&](int t) { return it.pair || (t & 1) == slot; };
                auto q_done = [&]() {  // two arrivals: this thread's twice, or each slot's once
                    pa_commit(&ctl->qempty[qt]);
                    if (it.pair || n == 1) pa_commit(&ctl->qempty[qt]);
                };
                for (int t = 0; t < D && t < n; ++t)
#pragma unroll
                    for (int h = 0; h < 2 && ok; ++h) {
                        if (mine(t)) score(h, qa);
                        else pass(false, t, h);
                    }
                const int first = it.pair ? 0 : slot;
                if (ok && first < n && first + D >= n) q_done();
                for (int t = 0; t < n && ok; ++t) {
                    const bool more = t + D < n, own = mine(t);
#pragma unroll
                    for (int h = 0; h < 2 && ok; ++h) {
                        if (own) value(t, h, t >= D, !more);
                        else pass(true, t, h);
                        if (more && ok) {
                            if (own) score(h, qa);
                            else pass(false, t + D, h);
                        }
                    }
                    if (own && more && t + 2 * D >= n && ok) q_done();
                }
                if (it.pair) {
                    ++nq[0];
                    ++nq[1];
                } else {
                    ++nq[qb];
                    qb ^= 1;
                }
                tiles += n;
            }
            // every MMA issued above has completed before the tensor memory is released
            pa_commit(&ctl->done);
            if (!mbar_wait(&ctl->done, 0)) set_dev_error(p.err, DEV_ERR_FULL_WAIT);
        }
        __syncwarp();
    } else if (warp == 10) {
        // ---------------- V rows that no row of the item may see become zero ----------------
        const int vbox = min(ps, kPaKeys / 2);
        for (uint32_t r = 0;; ++r) {
            // no request may come for long; the TMA warp always posts the last one, and itself waits for 2 s at most
            bool there = false;
            for (int n = 0; n < 1024 && !there && !*(volatile int*)&ctl->abort; ++n)
                there = __all_sync(0xffffffffu, mbar_wait(&ctl->fq[r & 15], r >> 4 & 1));
            if (!there) break;
            const int4 f = ctl->fix[r & 15];
            if (f.x < 0 || !pa_wait_warp(&ctl->full[f.x], f.y, ctl, p.err, DEV_ERR_FULL_WAIT)) break;
            const int hi = f.w & 0xFFFF;
            // 8 lanes a row (16 bytes each of 128), 4 rows at a time
            for (int q = lane >> 3; q < 64; q += 4)
                if (q < f.z || q >= hi || !(f.w >> (16 + (q >> 4)) & 1))
                    for (int h = 0; h < NH; ++h)
                        asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(kvs + f.x * STAGE + (q / vbox * NH + h) * vbox * 128 + q % vbox * 128 + (lane & 7) * 16),
                                     "r"(0)
                                     : "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctl->fixed[f.x]);
        }
    } else {
        // ---------------- softmax: thread = row of its slot ----------------
        const int slot = warp >> 2, row = tid & 127;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts0 = tmem + lanes + slot * 128, to = tmem + lanes + 256 + slot * HD;
        const int row_tok = row / G, row_head = row - row_tok * G;
        const float kLog2e = 1.4426950408889634f;
        const float sc2 = a.scale * kLog2e;
        // capped: cap log2e tanh(x) with x = scale s / cap, as cap log2e (1 - 2 / (1 + 2^(2 log2e x)))
        const float cap2 = a.softcap * kLog2e, x1 = a.softcap > 0.f ? a.scale / a.softcap : 0.f;
        const CapPoly kcap = cap_poly(cap2);
        uint32_t ns = 0, np = 0, nd = 0, nm = 0, tiles = 0;  // phases of sfull, ofull, odone and the merges; key tiles so far
        bool ok = true;
        for (int k = 0; ok; ++k) {
            PaItem it;
            if (!pa_next(ctl, k, lane, p.err, it)) break;
            const int tok = it.tok0 + (it.pair ? slot * p.TPT : 0) + row_tok;
            const int head = it.kvh * G + row_head;
            const bool live = row_tok < p.TPT && tok < it.tok0 + it.ntok;
            // the row's own position, and its visible keys in the prefix and in its own positions
            int own = -1;
            if (live) {
                if (it.b >= 0) {
                    own = it.base + (tok - it.q0);
                } else {
                    own = 0;
                    if (a.window > 0 || a.alibi) {
                        const int b = pa_request(a, tok);
                        own = pa_kv(a, b) - pa_q(a, b) + (tok - a.q_start[b]);
                    }
                }
            }
            const int P = a.prefix_len, W = a.window;
            // lanes without a row see everything, so that they call for no masking; nothing reads what they compute
            const bool seeing = own >= 0;
            const int lo_o = W > 0 && live ? max(0, own + 1 - W) : 0, hi_o = !live ? INT32_MAX : seeing ? own + 1 : 0;
            const int lo_p = W > 0 && live ? max(0, P + own + 1 - W) : 0, hi_p = !live ? INT32_MAX : seeing ? P : 0;
            const float slope = MOD && a.alibi && live ? a.alibi[head] * kLog2e : 0.f;
            // a warp without a row of the item lets its rows' products run on whatever S holds: nothing reads them
            const bool idle = !__any_sync(0xffffffffu, live);
            float m = -INFINITY, l = 0.f;
            const int step = it.pair ? 1 : 2;
            uint32_t no = 0;  // products of this item
            for (int t = it.pair ? 0 : slot; t < it.n && ok; t += step, ++ns) {
                const PaTile kt = pa_tile(p, it, t);
#pragma unroll 1
                for (int h = 0; h < 2; ++h) {
                    ok = pa_wait_warp(&ctl->sfull[slot][h], ns & 1, ctl, p.err, DEV_ERR_FULL_WAIT);
                    if (!ok) break;
                    if (!idle) {
                        pa_fence_after();
                        const uint32_t ts = ts0 + h * 64;
                        uint32_t y[2][32];
                        pa_ld32(ts, y[0]);
                        pa_ld32(ts + 32, y[1]);
                        const int k0 = kt.k0 + h * 64;
                        const int lo = (kt.prefix ? lo_p : lo_o) - k0, hi = (kt.prefix ? hi_p : hi_o) - k0;
                        const uint32_t mask = *(volatile uint32_t*)&ctl->okmask[(tiles + t) & 15][h] & 0xFu;
                        const bool whole = __all_sync(0xffffffffu, lo <= 0 && hi >= 64 && mask == 0xFu);
                        pa_wait_ld(y[0]);
                        pa_wait_ld(y[1]);
                        if (MOD) {
                            if (a.softcap > 0.f) {
                                // scores below half the cap (nearly all): tanh without the special function unit, which
                                // the weights' exp2 already fills
                                float big = 0.f;
#pragma unroll
                                for (int c = 0; c < 2; ++c)
#pragma unroll
                                    for (int e = 0; e < 32; e += 2)
                                        big = fmaxf(big, fmaxf(fabsf(__uint_as_float(y[c][e])), fabsf(__uint_as_float(y[c][e + 1]))));
                                if (__all_sync(0xffffffffu, big * fabsf(x1) <= 0.5f)) {
#pragma unroll
                                    for (int c = 0; c < 2; ++c)
#pragma unroll
                                        for (int e = 0; e < 32; e += 2) {
                                            const float2 z = cap_small(__fmul2_rn(make_float2(__uint_as_float(y[c][e]), __uint_as_float(y[c][e + 1])),
                                                                                  make_float2(x1, x1)), kcap);
                                            y[c][e] = __float_as_uint(z.x);
                                            y[c][e + 1] = __float_as_uint(z.y);
                                        }
                                } else {  // the same choice for each score, whatever its neighbours are
#pragma unroll
                                    for (int c = 0; c < 2; ++c)
#pragma unroll
                                        for (int e = 0; e < 32; e += 2) {
                                            const float2 x = __fmul2_rn(make_float2(__uint_as_float(y[c][e]), __uint_as_float(y[c][e + 1])),
                                                                        make_float2(x1, x1));
                                            float2 z = cap_small(x, kcap);
                                            if (!(fabsf(x.x) <= 0.5f)) z.x = fmaf(rcp(1.f + ex2(x.x * (2.f * kLog2e))), -2.f * cap2, cap2);
                                            if (!(fabsf(x.y) <= 0.5f)) z.y = fmaf(rcp(1.f + ex2(x.y * (2.f * kLog2e))), -2.f * cap2, cap2);
                                            y[c][e] = __float_as_uint(z.x);
                                            y[c][e + 1] = __float_as_uint(z.y);
                                        }
                                }
                            }
                            // z = (capped, or scale log2e s) - slope distance, the distance of key e being (own - k0) - e
                            if (a.alibi || !(a.softcap > 0.f)) {
                                const float bias = slope * (float)((kt.prefix ? P : 0) + own - k0);
                                const float f = a.softcap > 0.f ? 1.f : sc2;
                                const float2 f2 = make_float2(f, f), s2 = make_float2(slope, slope), b2 = make_float2(-bias, -bias);
#pragma unroll
                                for (int c = 0; c < 2; ++c)
#pragma unroll
                                    for (int e = 0; e < 32; e += 2) {
                                        const float2 add = __ffma2_rn(s2, make_float2((float)(c * 32 + e), (float)(c * 32 + e + 1)), b2);
                                        const float2 z = __ffma2_rn(make_float2(__uint_as_float(y[c][e]), __uint_as_float(y[c][e + 1])), f2, add);
                                        y[c][e] = __float_as_uint(z.x);
                                        y[c][e + 1] = __float_as_uint(z.y);
                                    }
                            }
                        }
                        if (!whole) {
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                // these 32 keys: bits [lo, hi) of those that were loaded
                                const int l0 = min(max(lo - c * 32, 0), 32), h0 = min(max(hi - c * 32, 0), 32);
                                uint32_t vis = (h0 < 32 ? (1u << h0) - 1u : 0xffffffffu) & ~(l0 < 32 ? (1u << l0) - 1u : 0xffffffffu);
                                if (!(mask >> (2 * c) & 1)) vis &= 0xffff0000u;
                                if (!(mask >> (2 * c + 1) & 1)) vis &= 0x0000ffffu;
#pragma unroll
                                for (int e = 0; e < 32; ++e)
                                    if (!(vis & (1u << e))) y[c][e] = 0xff800000u;  // -infinity
                            }
                        }
                        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                        for (int c = 0; c < 2; ++c)
#pragma unroll
                            for (int e = 0; e < 32; e += 2)
                                mx[(e >> 1) & 3] = fmaxf(mx[(e >> 1) & 3], fmaxf(__uint_as_float(y[c][e]), __uint_as_float(y[c][e + 1])));
                        float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                        if (!MOD) top *= sc2;
                        const bool rise = top > m + kSlack || (m == -INFINITY && top != -INFINITY);
                        if (__any_sync(0xffffffffu, rise)) {
                            const float factor = rise ? ex2(m - top) : 1.f;  // 0 from a maximum of -infinity
                            if (rise) m = top;
                            l *= factor;
                            if (no > 0) {
                                // O of the keys so far refers to the old maximum
                                ok = pa_wait_warp(&ctl->ofull[slot], (np + no - 1) & 1, ctl, p.err, DEV_ERR_FULL_WAIT);
                                if (!ok) break;
                                pa_fence_after();
#pragma unroll 1
                                for (int c = 0; c < HD / 32; ++c) {
                                    uint32_t o[32];
                                    pa_ld32(to + c * 32, o);
                                    pa_wait_ld(o);
#pragma unroll
                                    for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
                                    pa_st32(to + c * 32, o);
                                }
                            }
                        }
                        const float ref = (m == -INFINITY ? 0.f : m) - kShift;
                        const float2 ref2 = make_float2(-ref, -ref), one2 = make_float2(MOD ? 1.f : sc2, MOD ? 1.f : sc2);
                        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                        uint32_t pk[32];
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            float2 z = __ffma2_rn(make_float2(__uint_as_float(y[e >> 4][(e & 15) * 2]), __uint_as_float(y[e >> 4][(e & 15) * 2 + 1])),
                                                  one2, ref2);
                            z.x = ex2(z.x);
                            z.y = ex2(z.y);
                            sum[e & 1] = __fadd2_rn(sum[e & 1], z);
                            pk[e] = pa_pack<T>(z.x, z.y);
                        }
                        pa_st32(ts, pk);
                        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                        pa_wait_st();
                        pa_fence_before();
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ctl->pready[slot][h]);
                    ++no;
                }
            }
            if (!ok) break;
            tiles += it.n;
            // ---- the item's result ----
            if (no > 0) {
                ok = pa_wait_warp(&ctl->odone[slot], nd & 1, ctl, p.err, DEV_ERR_FULL_WAIT);
                if (!ok) break;
                pa_fence_after();
                ++nd;
            }
            np += no;
            float f0 = 1.f, f1 = 0.f;
            const bool merge = !it.pair && it.n > 1;
            if (merge) {
                if (slot == 1) {
                    ctl->ml1[row] = make_float2(m, l);
                    pa_fence_before();
                    mbar_arrive(&ctl->mready);
                } else {
                    ok = pa_wait_warp(&ctl->mready, nm & 1, ctl, p.err, DEV_ERR_FULL_WAIT);
                    if (!ok) break;
                    pa_fence_after();
                    const float2 other = ctl->ml1[row];
                    const float mm = fmaxf(m, other.x), mr = mm == -INFINITY ? 0.f : mm;
                    f0 = ex2(m - mr);
                    f1 = ex2(other.x - mr);
                    m = mm;
                    l = l * f0 + other.y * f1;
                }
            }
            if ((it.pair || slot == 0) && !idle) {
                const size_t ld = (size_t)a.n_tokens * a.n_heads;
                const size_t prow = ((size_t)it.kvh * a.n_tokens + tok) * G + row_head;
                const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // NaN stays NaN
#pragma unroll 1
                for (int c = 0; c < HD / 32; ++c) {
                    uint32_t o[32];
                    if (it.n > 0) {
                        pa_ld32(to + c * 32, o);
                        pa_wait_ld(o);
                        if (merge) {
                            uint32_t o1[32];
                            pa_ld32(to + HD + c * 32, o1);
                            pa_wait_ld(o1);
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                o[e] = __float_as_uint(__uint_as_float(o[e]) * f0 + __uint_as_float(o1[e]) * f1);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = 0u;
                    }
                    if (!live) continue;
                    if (it.direct) {
                        uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (size_t)tok * a.out_ld + (size_t)head * a.out_head + c * 32);
                        uint32_t pk[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            pk[e] = pa_pack<T>(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
#pragma unroll
                        for (int e = 0; e < 4; ++e) dst[e] = make_uint4(pk[4 * e], pk[4 * e + 1], pk[4 * e + 2], pk[4 * e + 3]);
                    } else {
                        float4* dst = p.acc + ((size_t)it.split * (HD / 4) + c * 8) * ld + prow;
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            dst[e * ld] = make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]), __uint_as_float(o[4 * e + 2]),
                                                 __uint_as_float(o[4 * e + 3]));
                    }
                }
                if (!it.direct && live) p.ml[it.split * ld + prow] = make_float2(m, l);
            }
            if (merge) {
                if (slot == 0) {
                    pa_fence_before();
                    mbar_arrive(&ctl->mdone);
                } else {
                    ok = pa_wait_warp(&ctl->mdone, nm & 1, ctl, p.err, DEV_ERR_FULL_WAIT);
                    if (!ok) break;
                }
                ++nm;
            }
        }
    }
    pa_fence_before();
    __syncthreads();
    pa_fence_after();
    if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// ---------------------------------------------------------------------------------------------
// Few rows: every request of the call has at most 16 query rows per kv head (decode, short verifies).  Reading the
// request's own K/V bounds it, so the small MMAs of mma.sync do, three CTAs share an SM and hide each other's latencies,
// and 16-byte asynchronous copies fetch a page of any size equally well (a TMA box of 16 rows is dear, see k_pattn).
// 64 contexts of 4096, 32 / 8 heads of 128, pages of 16: 8 rows 188 us (5.7 TB/s), 16 rows 204 us against 271 us by
// k_pattn (203 against 204 with pages of 128); at 20 rows it would take 306 us against 274, so 16 is the limit.  Two stages
// of 64 keys and three CTAs took 193 us at 64 ragged contexts up to 8192, three stages and two CTAs 235 us.
//
// A CTA has one (kv head, chunk, request); four warps take 16 of each 64 keys.  S^T = K Q^T (keys x rows) and
// O^T = V^T P^T (dims x rows), rows in NT tiles of 8, so nothing is padded to 128 rows; each warp keeps its own running
// (max, sum, O), joined at the end.  Keys that no row sees are fetched as zeros.
// ---------------------------------------------------------------------------------------------
constexpr int kRwThreads = 128, kRwKeys = 64, kRwStages = 2, kRwMaxRows = 16;
template <int HD> constexpr int rw_ld() { return HD + 8; }  // padded row of shared memory: ldmatrix without conflicts
template <int HD, int NT>
constexpr size_t rw_smem() {
    return ((size_t)NT * 8 + kRwStages * 2 * kRwKeys) * rw_ld<HD>() * 2;
}

__device__ __forceinline__ void rw_cp16(uint32_t dst, const void* src, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16u : 0u) : "memory");
}
__device__ __forceinline__ void rw_ldsm2(uint32_t a, uint32_t& x, uint32_t& y) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0, %1}, [%2];" : "=r"(x), "=r"(y) : "r"(a) : "memory");
}
__device__ __forceinline__ void rw_ldsm4(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ void rw_ldsm4t(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ uint32_t rw_transpose(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <class T>
__device__ __forceinline__ void rw_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <class T, int HD, int NT>
__global__ void __launch_bounds__(kRwThreads) k_pattn_rows(const __grid_constant__ PaArgs p) {
    constexpr bool BF = !std::is_same<T, __half>::value;
    constexpr float kShift = BF ? 0.f : 6.f, kSlack = 8.f;  // as in k_pattn
    constexpr int LD = rw_ld<HD>(), CPR = HD / 8, KPP = kRwThreads / CPR;  // 16-byte pieces per row, keys per pass
    extern __shared__ __align__(16) uint8_t rsm[];
    const sd_attn_args& a = p.a;
    const int kvh = blockIdx.x, c = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int n_tok = pa_rows(a, b), q = pa_q(a, b), kv = pa_kv(a, b), G = p.G, W = a.window;
    if (kvh == 0 && c == 0 && tid == 0 &&
        (a.q_len[b] > a.max_q || a.q_len[b] < 0 || a.kv_len[b] > a.max_kv || a.kv_len[b] < 0 || a.q_start[b] < 0 || n_tok < q))
        set_dev_error(p.err, DEV_ERR_BAD_ARG);
    pdl_trigger();
    if (n_tok == 0) return;
    int size;
    const int chunks = pa_chunks(p, kv, false, &size);
    if (c >= chunks) return;
    const int q0 = max(a.q_start[b], 0), base = kv - q, nrow = n_tok * G;
    // the last chunk's end would pass 32 bits in the longest contexts
    const int hi = min(max(base + n_tok, 0), c + 1 < chunks ? (c + 1) * size * kPaKeys : kv), lo = W > 0 ? max(0, base + 1 - W) : 0;
    const int first = max(c * size * kPaKeys, lo & ~(kRwKeys - 1));
    const int n = first < hi ? (hi - first + kRwKeys - 1) / kRwKeys : 0;
    T* qsm = reinterpret_cast<T*>(rsm);
    T* ring = qsm + NT * 8 * LD;
    const int ps = a.pool.page_size, lps = 31 - __clz(ps);
    const int32_t* table = a.table + (size_t)b * a.table_ld;

    // this thread's pieces of a stage: elements d8.. of keys key0 + KPP i
    const int d8 = (tid % CPR) * 8, key0 = tid / CPR;
    const T* kp = static_cast<const T*>(a.pool.k) + (size_t)kvh * a.pool.head_stride + d8;
    const T* vp = static_cast<const T*>(a.pool.v) + (size_t)kvh * a.pool.head_stride + d8;
    int ids[4];  // pages of the next stage's 16-key groups
    auto load_ids = [&](int s) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = first + s * kRwKeys + 16 * j;
            ids[j] = s < n && k < hi && k + 16 > lo ? table[k >> lps] : -2;
        }
    };
    uint32_t masks = 0;  // 4 bits per stage: groups that are there; the latest issued lowest
    auto issue = [&](int s) {
        if (s < n) {
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool have = ids[j] >= 0 && ids[j] < a.pool.n_pages;
                if (!have && ids[j] != -2 && tid == 0) set_dev_error(p.err, DEV_ERR_BAD_ARG);
                m |= (uint32_t)have << j;
            }
            masks = masks << 4 | m;
            const uint32_t dst = smem_u32(ring + (size_t)(s % kRwStages) * 2 * kRwKeys * LD + key0 * LD + d8);
#pragma unroll
            for (int i = 0; i < kRwKeys / KPP; ++i) {
                const int r = key0 + i * KPP, k = first + s * kRwKeys + r, j = (i * KPP) >> 4;
                // KPP <= 16 divides 16: a pass lies in one group
                const bool ok = (m >> j & 1) && k < hi && k >= lo;
                const size_t at = ok ? (size_t)ids[j] * a.pool.page_stride + (size_t)(k & (ps - 1)) * a.pool.pos_stride : 0;
                rw_cp16(dst + i * KPP * LD * 2, kp + at, ok);
                rw_cp16(dst + (kRwKeys + i * KPP) * LD * 2, vp + at, ok);
            }
        } else {
            masks <<= 4;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    load_ids(0);
#pragma unroll
    for (int s = 0; s < kRwStages - 1; ++s) {
        issue(s);
        load_ids(s + 1);
    }
    // Q rows (token, head of the group), zero behind them
    for (int i = tid; i < NT * 8 * CPR; i += kRwThreads) {
        const int r = i / CPR, d = (i - r * CPR) * 8;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (r < nrow) {
            const int t = r / G, h = r - t * G;
            x = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + (size_t)(q0 + t) * a.q_ld + (size_t)(kvh * G + h) * a.q_head + d);
        }
        *reinterpret_cast<uint4*>(qsm + r * LD + d) = x;
    }
    // the rows whose scores this thread holds: 8 nt + 2 (lane % 4) + e
    const int g = lane >> 2, t4 = lane & 3, lr = lane & 7, lq = lane >> 3;
    int end[NT][2];  // first key that the row does not see
    float slope[NT][2];
    const float kLog2e = 1.4426950408889634f, sc2 = a.scale * kLog2e;
    const float cap2 = a.softcap * kLog2e, x1 = a.softcap > 0.f ? a.scale / a.softcap : 0.f;
    const CapPoly kcap = cap_poly(cap2);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = nt * 8 + 2 * t4 + e, t = r / G;
            end[nt][e] = r < nrow ? max(base + t + 1, 0) : 0;
            slope[nt][e] = a.alibi && r < nrow ? a.alibi[kvh * G + r - t * G] * kLog2e : 0.f;
        }
    float m[NT][2], l[NT][2], o[HD / 16][NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) m[nt][e] = -INFINITY, l[nt][e] = 0.f;
#pragma unroll
    for (int i = 0; i < HD / 16; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][nt][e] = 0.f;
    const uint32_t q_a = smem_u32(qsm + lr * LD + (lq & 1) * 8);
    const uint32_t k_off = ((warp * 16 + lr + (lq & 1) * 8) * LD + (lq >> 1) * 8) * 2;
    const uint32_t v_off = ((kRwKeys + warp * 16 + lr + (lq >> 1) * 8) * LD + (lq & 1) * 8) * 2;
    for (int s = 0; s < n; ++s) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kRwStages - 2) : "memory");
        __syncthreads();  // stage s is there for everyone; the one before it is free
        issue(s + kRwStages - 1);
        load_ids(s + kRwStages);
        const uint32_t st = smem_u32(ring + (size_t)(s % kRwStages) * 2 * kRwKeys * LD);
        float sc[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) {
            uint32_t kf[4];
            rw_ldsm4(st + k_off + ks * 32, kf);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                uint32_t b0, b1;
                rw_ldsm2(q_a + (nt * 8 * LD + ks * 16) * 2, b0, b1);
                rw_mma<T>(sc[nt], kf, b0, b1);
            }
        }
        const int kg = first + s * kRwKeys + warp * 16 + g;  // this thread's keys: kg and kg + 8
        const bool there = masks >> (4 * (kRwStages - 1) + warp) & 1;
        uint32_t pf[NT][2];
        float fac[NT][2];
        bool rise = false;
        if (a.softcap > 0.f) {
            // as in k_pattn, the same choice for each score whatever its neighbours are: the quotient's error is a part of
            // the cap, so small scores take the polynomial, whose error is a part of the score (and which is no slower: decode
            // of 64 ragged contexts 194.0 us, 195.4 with the quotient for all)
            float2 x[NT][2];
            bool big = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    x[nt][e] = __fmul2_rn(make_float2(sc[nt][2 * e], sc[nt][2 * e + 1]), make_float2(x1, x1));
                    const float2 z = cap_small(x[nt][e], kcap);
                    sc[nt][2 * e] = z.x;
                    sc[nt][2 * e + 1] = z.y;
                    big |= !(fabsf(x[nt][e].x) <= 0.5f) || !(fabsf(x[nt][e].y) <= 0.5f);
                }
            if (__any_sync(0xffffffffu, big)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float y = e & 1 ? x[nt][e >> 1].y : x[nt][e >> 1].x;
                        if (!(fabsf(y) <= 0.5f)) sc[nt][e] = fmaf(rcp(1.f + ex2(y * (2.f * kLog2e))), -2.f * cap2, cap2);
                    }
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int k = kg + (e >> 1) * 8, stop = end[nt][e & 1];
                float z = a.softcap > 0.f ? sc[nt][e] : sc[nt][e] * sc2;
                if (a.alibi) z = fmaf(slope[nt][e & 1], (float)(k - (stop - 1)), z);
                if (!there || k >= stop || (W > 0 && k < stop - W)) z = -INFINITY;
                sc[nt][e] = z;
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float top = fmaxf(sc[nt][e], sc[nt][e + 2]);
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
                fac[nt][e] = 1.f;
                if (top > m[nt][e] + kSlack || (m[nt][e] == -INFINITY && top != -INFINITY)) {
                    fac[nt][e] = ex2(m[nt][e] - top);
                    m[nt][e] = top;
                    rise = true;
                }
                const float ref = (m[nt][e] == -INFINITY ? 0.f : m[nt][e]) - kShift;
                sc[nt][e] = ex2(sc[nt][e] - ref);
                sc[nt][e + 2] = ex2(sc[nt][e + 2] - ref);
                l[nt][e] = fmaf(l[nt][e], fac[nt][e], sc[nt][e] + sc[nt][e + 2]);
            }
            pf[nt][0] = rw_transpose(pa_pack<T>(sc[nt][0], sc[nt][1]));
            pf[nt][1] = rw_transpose(pa_pack<T>(sc[nt][2], sc[nt][3]));
        }
        if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
            for (int i = 0; i < HD / 16; ++i)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[i][nt][e] *= fac[nt][e & 1];
        }
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
            uint32_t vf[4];
            rw_ldsm4t(st + v_off + i * 32, vf);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) rw_mma<T>(o[i][nt], vf, pf[nt][0], pf[nt][1]);
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();  // the ring becomes the warps' states: O [warp][row][dim], (max, sum) [warp][row]
    constexpr int OLD = HD + 4;
    float* osm = reinterpret_cast<float*>(ring);
    float2* msm = reinterpret_cast<float2*>(osm + 4 * NT * 8 * OLD);
    static_assert((size_t)4 * NT * 8 * (OLD * 4 + 8) <= (size_t)kRwStages * 2 * kRwKeys * LD * 2, "the states fit the ring");
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], off);
#pragma unroll
        for (int i = 0; i < HD / 16; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) osm[(warp * NT * 8 + nt * 8 + 2 * t4 + (e & 1)) * OLD + i * 16 + g + (e >> 1) * 8] = o[i][nt][e];
        if (g == 0) {
            msm[warp * NT * 8 + nt * 8 + 2 * t4] = make_float2(m[nt][0], l[nt][0]);
            msm[warp * NT * 8 + nt * 8 + 2 * t4 + 1] = make_float2(m[nt][1], l[nt][1]);
        }
    }
    __syncthreads();
    const bool direct = chunks == 1 && a.prefix_len == 0;
    const size_t ld = (size_t)a.n_tokens * a.n_heads;
    for (int i = tid; i < nrow * (HD / 4); i += kRwThreads) {
        // neighbouring threads: neighbouring rows of the workspace, or neighbouring dims of the output
        const int r = direct ? i / (HD / 4) : i % nrow, d4 = direct ? i % (HD / 4) : i / nrow;
        float M = -INFINITY, L = 0.f;
        float2 ml[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            ml[w] = msm[w * NT * 8 + r];
            M = fmaxf(M, ml[w].x);
        }
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = ml[w].x == -INFINITY && ml[w].y == 0.f ? 0.f : ex2(ml[w].x - M);
            const float4 y = *reinterpret_cast<const float4*>(osm + (w * NT * 8 + r) * OLD + d4 * 4);
            L = fmaf(ml[w].y, f, L);
            x.x = fmaf(y.x, f, x.x);
            x.y = fmaf(y.y, f, x.y);
            x.z = fmaf(y.z, f, x.z);
            x.w = fmaf(y.w, f, x.w);
        }
        const int t = r / G, h = r - t * G;
        if (direct) {
            const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
            T* dst = static_cast<T*>(a.out) + (size_t)(q0 + t) * a.out_ld + (size_t)(kvh * G + h) * a.out_head + d4 * 4;
            *reinterpret_cast<uint2*>(dst) = make_uint2(pa_pack<T>(x.x * inv, x.y * inv), pa_pack<T>(x.z * inv, x.w * inv));
        } else {
            const size_t prow = ((size_t)kvh * a.n_tokens + q0 + t) * G + h;
            p.acc[((size_t)(p.cp + c) * (HD / 4) + d4) * ld + prow] = x;
            if (d4 == 0) p.ml[(size_t)(p.cp + c) * ld + prow] = make_float2(M, L);
        }
    }
}

// Joins the states that the items of a row left: o = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i, in split order.
// lane = row, warp = 4 DV of the dims, so the states are read in whole lines, several splits' at a time.  It starts while
// the items still run (programmatic launch) and finds its rows' requests meanwhile.  DV = 4 reads each (max, sum) least
// often; with few rows DV = 1 gives the SMs four times the warps (1024 rows of 23 splits: 36 -> 11 us).
constexpr int kPaJoinWarps = 4;
template <class T, int HD, int DV>
__global__ void __launch_bounds__(kPaJoinWarps * 32) k_pattn_combine(const __grid_constant__ PaArgs p) {
    constexpr int U = DV == 1 ? 8 : 4;
    const sd_attn_args& a = p.a;
    const int lane = threadIdx.x & 31, d0 = (blockIdx.y * kPaJoinWarps + (threadIdx.x >> 5)) * 4 * DV;
    const size_t ld = (size_t)a.n_tokens * a.n_heads, row = (size_t)blockIdx.x * 32 + lane;
    const int gt = (int)min(row, ld - 1) / p.G, tok = gt % a.n_tokens, kvh = gt / a.n_tokens;
    const int head = kvh * p.G + (int)(row - (size_t)gt * p.G);
    const int b = pa_request(a, tok), t = tok - a.q_start[b], rows = pa_rows(a, b);
    const int kv = pa_kv(a, b);
    const bool inl = pa_inline(p, rows);
    int size;
    const int chunks = pa_chunks(p, kv, inl, &size);
    // else: no row, or written by its item
    const bool mine = row < ld && t >= 0 && t < rows && !(chunks == 1 && (a.prefix_len == 0 || inl));
    const bool seeing = mine && kv - pa_q(a, b) + t >= 0;
    const int s0 = inl ? p.cp : 0, s1 = seeing ? p.cp + chunks : s0;
    pdl_wait();
    if (!__any_sync(0xffffffffu, mine)) return;
    float M = -INFINITY;
#pragma unroll 8
    for (int s = s0; s < s1; ++s) M = fmaxf(M, p.ml[s * ld + row].x);
    if (M == -INFINITY) M = 0.f;
    float L = 0.f;
    float4 o[DV];
#pragma unroll
    for (int e = 0; e < DV; ++e) o[e] = make_float4(0.f, 0.f, 0.f, 0.f);
    const float4* acc = p.acc + (size_t)(d0 / 4) * ld + row;
    for (int c = s0; c < s1; c += U) {
        float2 ml[U];
        float4 x[U][DV];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = min(c + u, s1 - 1);
            ml[u] = p.ml[s * ld + row];
#pragma unroll
            for (int e = 0; e < DV; ++e) x[u][e] = acc[((size_t)s * (HD / 4) + e) * ld];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (c + u >= s1 || ml[u].y == 0.f) continue;  // a split that saw nothing has no O
            const float f = ex2(ml[u].x - M);
            L = fmaf(ml[u].y, f, L);
#pragma unroll
            for (int e = 0; e < DV; ++e) {
                o[e].x = fmaf(x[u][e].x, f, o[e].x);
                o[e].y = fmaf(x[u][e].y, f, o[e].y);
                o[e].z = fmaf(x[u][e].z, f, o[e].z);
                o[e].w = fmaf(x[u][e].w, f, o[e].w);
            }
        }
    }
    if (!mine) return;
    const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
    uint2* dst = reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (size_t)tok * a.out_ld + (size_t)head * a.out_head + d0);
#pragma unroll
    for (int e = 0; e < DV; ++e) dst[e] = make_uint2(pa_pack<T>(o[e].x * inv, o[e].y * inv), pa_pack<T>(o[e].z * inv, o[e].w * inv));
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
    static EncodeTiled fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<EncodeTiled>(f);
    }();
    return fn;
}

// What TMA and 16-byte accesses need, and a scale / cap that 32 bits hold in full (the scores are multiplied by it at once);
// other calls take the general kernel.
bool tc_able(const sd_attn_args& a) {
    const sd_kv_pool& k = a.pool;
    if (a.softcap > 0.f && a.scale != 0.f && !(std::fabs(a.scale / a.softcap) >= FLT_MIN)) return false;
    auto al = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
    auto st = [](int64_t s) { return s > 0 && s % 8 == 0 && s < (1ll << 38); };
    return (k.head_dim == 64 || k.head_dim == 128) && al(k.k) && al(k.v) && al(a.q) && al(a.out) && st(k.page_stride) &&
           st(k.pos_stride) && st(k.head_stride) && st(a.q_ld) && st(a.q_head) && st(a.out_ld) && st(a.out_head);
}

// How the work of a call is cut: depends on what the host knows only (counts and bounds), so a request's split
// does not depend on the other requests' kv_len.
void pa_plan(const sd_attn_args& a, int sms, PaArgs* p) {
    p->a = a;
    p->G = a.n_heads / a.pool.n_kv_heads;
    p->TPT = 128 / p->G;
    const int n_kv = a.pool.n_kv_heads, pair = 2 * p->TPT;
    p->np = (a.prefix_len + kPaKeys - 1) / kPaKeys;
    const int own = (a.max_kv + kPaKeys - 1) / kPaKeys + (a.max_q > pair ? p->np : 0);
    const long long units = (long long)n_kv * std::max<long long>(a.n_req, a.n_tokens / pair);
    // tiles that an item can see through the window; if those fit one chunk, nothing is cut
    const int seen = a.window > 0 ? (int)std::min<long long>(own, ((long long)a.window + std::min(a.max_q, pair)) / kPaKeys + 2) : own;
    int ct = std::max(seen, 1);
    p->few = (long long)a.max_q * p->G <= kRwMaxRows;
    if (p->few) {
        // a chunk costs about a tile to start and to join; the kernel keeps several CTAs on an SM
        ct = std::max(1, (int)(std::sqrt((double)units * seen / (2.0 * sms)) + 0.5));
    } else if (a.max_q <= p->TPT) {
        // few rows per item: a chunk costs about one tile to start and to join, and the last one to end leaves the
        // other SMs idle for up to its length: the sum is least at the square root of an SM's tiles
        const double per_sm = (double)units * seen / sms;
        ct = std::max(4, (int)(std::sqrt(per_sm) + 0.5));
    } else {
        // many rows: whole rounds over the SMs, in key tiles of about 2.2 us.  A cut costs an item about 3 tiles more, and
        // the join reads and the items write O of every row in 32 bits once per split (about 4 TB/s; without that term
        // 8 prompts behind a prefix of 8192 were cut in two and took 477 us, uncut 439, in short bursts)
        const double join = (double)a.n_tokens * a.n_heads * (a.pool.head_dim * 8 + 16) / 4e12 / 2.2e-6;
        double best = 1e300;
        for (int n = 1; n <= 32; ++n) {
            const long long rounds = (units * n + sms - 1) / sms;
            const double t = (double)rounds * ((seen + n - 1) / n + 1.5 + (n > 1 ? 3.0 : 0.0)) + (n > 1 ? n * join : 0.0);
            if (t < best * 0.97) best = t, ct = (seen + n - 1) / n;
        }
    }
    p->ct_own = ct >= seen ? std::max(own, 1) : std::max(ct, 1);
    // prefix items: one round over the SMs
    p->n_pt = p->np ? (a.n_tokens + pair - 1) / pair : 0;
    p->ct_pre = 1;
    p->cp = 0;
    if (p->np) {
        const long long u = (long long)n_kv * p->n_pt;
        const long long n = std::max<long long>(1, std::min<long long>((p->np + 3) / 4, sms / u));
        p->ct_pre = (int)((p->np + n - 1) / n);
        p->cp = (p->np + p->ct_pre - 1) / p->ct_pre;
    }
}

int pa_splits(const PaArgs& p) {
    const sd_attn_args& a = p.a;
    const int own = (a.max_kv + kPaKeys - 1) / kPaKeys + (p.np && a.max_q > 2 * p.TPT ? p.np : 0);
    const int chunks = std::max(1, (own + p.ct_own - 1) / p.ct_own);
    return chunks == 1 && p.np == 0 ? 0 : p.cp + chunks;
}

size_t pa_workspace(const PaArgs& p) {
    const size_t rows = (size_t)pa_splits(p) * p.a.n_tokens * p.a.n_heads;
    return rows * ((size_t)p.a.pool.head_dim * 4 + 8);
}

int encode(CUtensorMap* m, bool bf16, int rank, const void* base, const cuuint64_t* dims, const cuuint64_t* strides,
           const cuuint32_t* box) {
    const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
    EncodeTiled fn = encode_tiled();
    if (!fn) return fail(SD_ERR_UNSUPPORTED, "cuTensorMapEncodeTiled is not available");
    const CUresult r = fn(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, const_cast<void*>(base),
                          dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? SD_OK : fail(SD_ERR_INVALID, "attention: tensor map refused (%d)", (int)r);
}

static_assert(pa_smem<128>(SD_PAGES_MAX_REQ) <= 232448, "the largest batch fits the shared memory");

template <class T, int HD, int NT>
int launch_rows(const PaArgs& p, int dev, cudaStream_t st) {
    static std::atomic<bool> ready[64];
    cudaError_t e = cudaSuccess;
    if (dev < 0 || dev >= 64 || !ready[dev].load(std::memory_order_acquire)) {
        e = cudaFuncSetAttribute(k_pattn_rows<T, HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)rw_smem<HD, NT>());
        if (e != cudaSuccess) return cuda_fail(e, "attention attributes");
        if (dev >= 0 && dev < 64) ready[dev].store(true, std::memory_order_release);
    }
    const int own = (p.a.max_kv + kPaKeys - 1) / kPaKeys;
    const int chunks = std::max(1, (own + p.ct_own - 1) / p.ct_own);
    if (chunks > 65535) return fail(SD_ERR_INVALID, "sd_attention_dev: too many work items");
    k_pattn_rows<T, HD, NT><<<dim3(p.a.pool.n_kv_heads, chunks, p.a.n_req), kRwThreads, rw_smem<HD, NT>(), st>>>(p);
    e = cudaGetLastError();
    return e == cudaSuccess ? SD_OK : cuda_fail(e, "attention");
}

template <class T, int HD, bool MOD>
int launch_tc(const PaArgs& p, int grid, int dev, cudaStream_t st) {
    const size_t smem = pa_smem<HD>(p.a.n_req);
    static std::atomic<bool> ready[64];  // per device: the largest batch's shared memory is allowed
    cudaError_t e = cudaSuccess;
    if (dev < 0 || dev >= 64 || !ready[dev].load(std::memory_order_acquire)) {
        e = cudaFuncSetAttribute(k_pattn<T, HD, MOD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)pa_smem<HD>(SD_PAGES_MAX_REQ));
        if (e != cudaSuccess) return cuda_fail(e, "attention attributes");
        if (dev >= 0 && dev < 64) ready[dev].store(true, std::memory_order_release);
    }
    if (grid > 0) {
        k_pattn<T, HD, MOD><<<grid, kPaThreads, smem, st>>>(p);
        if ((e = cudaGetLastError()) != cudaSuccess) return cuda_fail(e, "attention");
    }
    if (p.few) {
        const int rc = p.a.max_q * p.G <= 8 ? launch_rows<T, HD, 1>(p, dev, st) : launch_rows<T, HD, 2>(p, dev, st);
        if (rc) return rc;
    }
    if (pa_splits(p) > 0) {
        cudaLaunchConfig_t cfg{};
        const unsigned blocks = (unsigned)(((long long)p.a.n_tokens * p.a.n_heads + 31) / 32);
        const bool many = blocks >= (unsigned)device_sm_count(dev);
        cfg.gridDim = dim3(blocks, HD / 4 / kPaJoinWarps / (many ? 4 : 1));
        cfg.blockDim = dim3(kPaJoinWarps * 32);
        cfg.stream = st;
        cudaLaunchAttribute at{};
        at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at.val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = &at;
        cfg.numAttrs = 1;
        e = many ? cudaLaunchKernelEx(&cfg, k_pattn_combine<T, HD, 4>, p) : cudaLaunchKernelEx(&cfg, k_pattn_combine<T, HD, 1>, p);
        if (e != cudaSuccess) return cuda_fail(e, "attention combine");
    }
    return SD_OK;
}

int run_tc(const sd_attn_args& a, int dev, int* err, cudaStream_t st) {
    if ((long long)a.n_tokens * a.n_heads > INT32_MAX - 64) return fail(SD_ERR_INVALID, "sd_attention_dev: too many rows");
    PaArgs p{};
    pa_plan(a, device_sm_count(dev), &p);
    const size_t need = pa_workspace(p);
    if (need > 0 && (!a.workspace || a.workspace_bytes < need || (reinterpret_cast<uintptr_t>(a.workspace) & 255)))
        return fail(SD_ERR_INVALID, "sd_attention_dev: %zu bytes of 256-byte aligned workspace needed", need);
    const size_t rows = (size_t)pa_splits(p) * a.n_tokens * a.n_heads;
    p.acc = static_cast<float4*>(a.workspace);
    p.ml = reinterpret_cast<float2*>(p.acc + rows * (a.pool.head_dim / 4));
    p.err = err;
    const sd_kv_pool& k = a.pool;
    const bool bf = k.dtype == SD_BF16;
    const int pair = 2 * p.TPT;
    const int own = (a.max_kv + kPaKeys - 1) / kPaKeys + (p.np && a.max_q > pair ? p.np : 0);
    const long long items = (long long)k.n_kv_heads * ((long long)p.cp * p.n_pt + (p.few ? 0LL : (long long)a.n_req + a.n_tokens / pair) *
                                                       std::max(1, (own + p.ct_own - 1) / p.ct_own));
    if (items > INT32_MAX) return fail(SD_ERR_INVALID, "sd_attention_dev: too many work items");
    const int grid = (int)items;
    if (grid > 0) {  // k_pattn's tensor maps
        const cuuint64_t hd = k.head_dim;
        {
            const cuuint64_t dims[3] = {hd, (cuuint64_t)a.n_heads, (cuuint64_t)a.n_tokens};
            const cuuint64_t strides[2] = {(cuuint64_t)a.q_head * 2, (cuuint64_t)a.q_ld * 2};
            const cuuint32_t box[3] = {64, (cuuint32_t)p.G, (cuuint32_t)p.TPT};
            const int rc = encode(&p.tq, bf, 3, a.q, dims, strides, box);
            if (rc) return rc;
        }
        for (int i = 0; i < 2; ++i) {
            const cuuint32_t rows = std::min(k.page_size, kPaKeys / 2), nh = k.head_dim / 64;
            const cuuint64_t dims[5] = {64, (cuuint64_t)k.page_size, nh, (cuuint64_t)k.n_kv_heads, (cuuint64_t)k.n_pages};
            const cuuint64_t strides[4] = {(cuuint64_t)k.pos_stride * 2, 128, (cuuint64_t)k.head_stride * 2, (cuuint64_t)k.page_stride * 2};
            const cuuint32_t box[5] = {64, rows, i || rows == kPaKeys / 2 ? nh : 1, 1, 1};
            const int rc = encode(i ? &p.tv : &p.tk, bf, 5, i ? k.v : k.k, dims, strides, box);
            if (rc) return rc;
        }
    }
    const bool mod = a.softcap > 0.f || a.alibi || !(a.scale > 0.f);
    if (bf) {
        if (k.head_dim == 128) return mod ? launch_tc<__nv_bfloat16, 128, true>(p, grid, dev, st) : launch_tc<__nv_bfloat16, 128, false>(p, grid, dev, st);
        return mod ? launch_tc<__nv_bfloat16, 64, true>(p, grid, dev, st) : launch_tc<__nv_bfloat16, 64, false>(p, grid, dev, st);
    }
    if (k.head_dim == 128) return mod ? launch_tc<__half, 128, true>(p, grid, dev, st) : launch_tc<__half, 128, false>(p, grid, dev, st);
    return mod ? launch_tc<__half, 64, true>(p, grid, dev, st) : launch_tc<__half, 64, false>(p, grid, dev, st);
}

int check_attention(const sd_attn_args* a) {
    const char* what = "sd_attention_dev";
    if (!a) return fail(SD_ERR_INVALID, "%s: null arguments", what);
    int rc = check_kv_pool(&a->pool, what);
    if (rc) return rc;
    if ((a->n_tokens != 0 && (!a->q || !a->out)) || !a->table || !a->kv_len || !a->q_start || !a->q_len)
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
    if (!(std::fabs(a->scale) <= 1e30f) || !(a->softcap == 0.f || (a->softcap >= 1e-6f && a->softcap <= 1e30f)))
        return fail(SD_ERR_INVALID, "%s: scale %g, softcap %g", what, a->scale, a->softcap);
    if (a->q_head < a->pool.head_dim || a->out_head < a->pool.head_dim || a->q_ld < 0 || a->out_ld < 0)
        return fail(SD_ERR_INVALID, "%s: strides", what);
    if (a->n_tokens > 1 && a->out_ld < a->pool.head_dim) return fail(SD_ERR_INVALID, "%s: the tokens of out overlap", what);
    return SD_OK;
}

}  // namespace

int launch_paged_attention(const sd_attn_args* a, int dev, int* err, cudaStream_t st) {
    if (tc_able(*a)) return run_tc(*a, dev, err, st);
    const long long rows = (long long)a->n_tokens * a->n_heads;
    if ((rows + 3) / 4 > INT32_MAX) return fail(SD_ERR_INVALID, "sd_attention_dev: too many rows");
    const int grid = (int)((rows + 3) / 4);
    if (a->pool.dtype == SD_F16)
        k_pattn_general<__half><<<grid, 128, 0, st>>>(*a, err);
    else
        k_pattn_general<__nv_bfloat16><<<grid, 128, 0, st>>>(*a, err);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? SD_OK : cuda_fail(e, "attention");
}

}  // namespace sd

extern "C" {

size_t sd_attention_workspace(const sd_attn_args* a) {
    if (check_attention(a) || a->n_tokens == 0 || !tc_able(*a)) return 0;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) dev = 0;
    PaArgs p{};
    pa_plan(*a, device_sm_count(dev), &p);
    return pa_workspace(p);
}

int sd_attention_dev(const sd_attn_args* a, void* stream) {
    clear_error();
    int rc = check_attention(a), dev;
    if (rc) return rc;
    if (a->n_tokens == 0) return SD_OK;
    if ((rc = paged_device(a->pool.k, "sd_attention_dev", &dev))) return rc;
    return launch_paged_attention(a, dev, device_error_word(dev), (cudaStream_t)stream);
}

}  // extern "C"
