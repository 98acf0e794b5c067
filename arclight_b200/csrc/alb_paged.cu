// Paged K/V cache (sm_100a): appending the K/V rows of a batch of tokens with
// QK-norm and rotation on the way, and the attention of single query tokens
// over the pages.
#include <cmath>
#include <cuda_bf16.h>

#include "alb_common.cuh"
#include "alb_internal.h"

using namespace alb;

namespace {

// alb_paged_kv as the kernels take it: strides filled in, and the division of a
// position by page_size as one multiplication: for 0 <= n < 2^31 and
// s = ceil(log2 d), m = floor(2^32 (2^s - d) / d) + 1 gives
// n / d = (umulhi(n, m) + n) >> s (the round-up method; umulhi(n, m) + n < 2^32
// because umulhi(n, m) <= n < 2^31).
struct PagedView {
    uint16_t * k, * v;
    const int32_t * table;
    int64_t table_stride, page_stride, cell_stride, head_stride;
    int32_t n_pages, n_seqs, max_pages, page_size, Hkv;
    uint32_t div_mul, div_shift;
};

__device__ __forceinline__ int32_t page_of(const PagedView & kv, int32_t pos) {
    return (int32_t)((__umulhi((uint32_t)pos, kv.div_mul) + (uint32_t)pos) >> kv.div_shift);
}

// Element offset of a cell's head 0, or -1 when its page is out of range.
__device__ __forceinline__ int64_t cell_offset(const PagedView & kv, const int32_t * __restrict__ row, int32_t pos) {
    const int32_t p = page_of(kv, pos);
    const int32_t page = row[p];
    if ((uint32_t)page >= (uint32_t)kv.n_pages) return -1;
    return (int64_t)page * kv.page_stride + (int64_t)(pos - p * kv.page_size) * kv.cell_stride;
}

template <bool BF16> __device__ __forceinline__ uint16_t to_cache(float x) {
    if (BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(x));
    return alb_f2h(x);
}

template <int N> struct Vec;
template <> struct Vec<2> { using F = float2; };
template <> struct Vec<4> { using F = float4; };

// ------------------------------------------------------------------- append
// One warp per head of a token, N = D/32 neighbouring values per lane, so that
// the NEOX partner d +- D/2 of every value is the same slot of lane ^ 16.  The
// arithmetic is k_qk_norm_rope_kv's: fp32 squares summed in double (certified to
// round to the sequential sum's mean), then the fp32 products in its order.
template <int D, bool BF16>
__global__ void __launch_bounds__(256)
k_qk_norm_rope_kv_paged(const float * __restrict__ qkv, int64_t qkv_stride, int64_t n_items, int Hq,
                        const float * __restrict__ qn_w, const float * __restrict__ kn_w, float eps,
                        const float * __restrict__ rope, int32_t max_pos, const int32_t * __restrict__ positions,
                        const int32_t * __restrict__ seqs, PagedView kv, float * __restrict__ q_out, int * err) {
    constexpr int N = D / 32;
    using F = typename Vec<N>::F;
    const int lane = threadIdx.x & 31;
    const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    alb_pdl_wait();
    if (item >= n_items) { alb_pdl_trigger(); return; }   // (a whole warp; no block barrier follows)
    const int H = Hq + 2 * kv.Hkv;
    const int64_t t = item / H;
    const int head = (int)(item - t * H);
    const int32_t pos = positions[t];
    const int32_t seq = seqs ? seqs[t] : (t < kv.n_seqs ? (int32_t)t : kv.n_seqs);
    if (pos < 0 || seq < 0) { alb_pdl_trigger(); return; }
    const bool in_table = pos < max_pos && seq < kv.n_seqs && page_of(kv, pos) < kv.max_pages;
    const int64_t cell = in_table ? cell_offset(kv, kv.table + (int64_t)seq * kv.table_stride, pos) : -1;
    if (cell < 0) {
        if (lane == 0) atomicExch(err, ALB_DEVERR_BAD_INDEX);
        alb_pdl_trigger();
        return;
    }
    const float * src = qkv + t * qkv_stride + (int64_t)head * D;
    float x[N];
    *reinterpret_cast<F *>(x) = *reinterpret_cast<const F *>(src + N * lane);
    if (head < Hq + kv.Hkv) {
        const float * w = head < Hq ? qn_w : kn_w;
        if (w) {
            double s = 0.0;
#pragma unroll
            for (int i = 0; i < N; ++i) s += (double)__fmul_rn(x[i], x[i]);
            s = alb_warp_sum_d(s);
            if (!alb_rms_mean_certain(s, D)) {   // the reference's sequential sum (the whole warp)
                s = lane == 0 ? alb_rms_seq_sum(src, D) : 0.0;
                s = __shfl_sync(0xffffffffu, s, 0);
            }
            const float mean = (float)(s / (double)D);
            const float scale = 1.0f / sqrtf(__fadd_rn(mean, eps));
            float wv[N];
            *reinterpret_cast<F *>(wv) = *reinterpret_cast<const F *>(w + N * lane);
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = __fmul_rn(__fmul_rn(x[i], scale), wv[i]);
        }
        float cs[2 * N];
        const float * r = rope + (int64_t)pos * D + 2 * N * (lane & 15);
        *reinterpret_cast<F *>(cs) = *reinterpret_cast<const F *>(r);
        *reinterpret_cast<F *>(cs + N) = *reinterpret_cast<const F *>(r + N);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float y = __shfl_xor_sync(0xffffffffu, x[i], 16);
            x[i] = lane < 16 ? __fsub_rn(__fmul_rn(x[i], cs[2 * i]), __fmul_rn(y, cs[2 * i + 1]))
                             : __fadd_rn(__fmul_rn(y, cs[2 * i + 1]), __fmul_rn(x[i], cs[2 * i]));
        }
    }
    if (head < Hq) {
        *reinterpret_cast<F *>(q_out + (t * Hq + head) * D + N * lane) = *reinterpret_cast<F *>(x);
    } else {
        const bool is_k = head < Hq + kv.Hkv;
        const int h = head - Hq - (is_k ? 0 : kv.Hkv);
        uint16_t * dst = (is_k ? kv.k : kv.v) + cell + (int64_t)h * kv.head_stride + N * lane;
#pragma unroll
        for (int i = 0; i < N; i += 2)
            *reinterpret_cast<uint32_t *>(dst + i) =
                (uint32_t)to_cache<BF16>(x[i]) | ((uint32_t)to_cache<BF16>(x[i + 1]) << 16);
    }
    alb_pdl_trigger();
}

// ---------------------------------------------------------------- attention
template <bool BF16> __device__ __forceinline__ float from_cache(uint16_t h) {
    if (BF16) return __uint_as_float((uint32_t)h << 16);
    return alb_h2f(h);
}

// The plain form: one CTA per (query head, row), its four warps taking every
// fourth cell, a cell's D products spread over the lanes; online softmax per
// warp, the warps joined through shared memory.
template <int D, bool BF16>
__global__ void __launch_bounds__(128)
k_paged_attn(const float * __restrict__ q, int Hq, PagedView kv, const int32_t * __restrict__ seqs,
             const int32_t * __restrict__ lengths, int32_t window, float scale, float * __restrict__ out,
             float * __restrict__ lse, int * err) {
    constexpr int N = D / 32;
    const int64_t r = blockIdx.x;
    const int h = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __shared__ float sm[4], sl[4], so[4][D];
    alb_pdl_wait();
    int32_t len = lengths[r];
    if (len < 0) { alb_pdl_trigger(); return; }
    const int32_t seq = seqs ? seqs[r] : (r < kv.n_seqs ? (int32_t)r : -1);
    const int64_t most = (int64_t)kv.max_pages * kv.page_size;
    if (seq < 0 || seq >= kv.n_seqs || len > most) {
        if (threadIdx.x == 0) atomicExch(err, ALB_DEVERR_BAD_INDEX);
        len = seq < 0 || seq >= kv.n_seqs ? 0 : (int32_t)most;
    }
    const int32_t first = window > 0 && len > window ? len - window : 0;
    const int32_t * row = kv.table + (int64_t)(len ? seq : 0) * kv.table_stride;
    const int64_t head = (int64_t)(h / (Hq / kv.Hkv)) * kv.head_stride + N * lane;
    float qv[N], o[N], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) { qv[i] = q[(r * Hq + h) * D + N * lane + i]; o[i] = 0.0f; }
    for (int32_t j = first + warp; j < len; j += 4) {
        const int64_t cell = cell_offset(kv, row, j);
        if (cell < 0) {
            if (lane == 0) atomicExch(err, ALB_DEVERR_BAD_INDEX);
            continue;
        }
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) s = fmaf(qv[i], from_cache<BF16>(kv.k[cell + head + i]), s);
        s = alb_warp_sum(s) * scale;
        const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.0f : mn;
        const float c = expf(m - base), p = expf(s - base);
        l = fmaf(l, c, p);
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = fmaf(o[i], c, p * from_cache<BF16>(kv.v[cell + head + i]));
        m = mn;
    }
    if (lane == 0) { sm[warp] = m; sl[warp] = l; }
#pragma unroll
    for (int i = 0; i < N; ++i) so[warp][N * lane + i] = o[i];
    __syncthreads();
    const float M = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3])), base = M == -INFINITY ? 0.0f : M;
    float L = 0.0f, c[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) { c[w] = expf(sm[w] - base); L = fmaf(sl[w], c[w], L); }
    for (int d = threadIdx.x; d < D; d += 128) {
        float a = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) a = fmaf(so[w][d], c[w], a);
        out[(r * Hq + h) * D + d] = L != 0.0f ? a / L : 0.0f;
    }
    if (lse && threadIdx.x == 0) lse[r * Hq + h] = M + logf(L);
    alb_pdl_trigger();
}

// ------------------------------------------------------------------- checks
struct Axis { int64_t stride, count; };

// Fills the view; a message in alb_last_error() and false when the cache cannot
// be used.  The three strides must leave every cell a place of its own: sorted
// by stride, each axis spans no more than the next one's step.
bool paged_view(const alb_paged_kv * c, PagedView & kv, bool table) {
    const char * why = nullptr;
    if (!c) why = "invalid argument: the paged cache is NULL";
    else if (!c->k || !c->v || (table && !c->page_table)) why = "invalid argument: paged cache with a NULL pointer";
    else if (((uintptr_t)c->k | (uintptr_t)c->v) & 15) why = "invalid argument: paged cache k / v not 16-byte aligned";
    else if (c->head_dim != 64 && c->head_dim != 128) why = "invalid argument: paged cache head_dim is not 64 or 128";
    else if (c->type != ALB_KV_F16 && c->type != ALB_KV_BF16) why = "invalid argument: paged cache type";
    else if (c->n_pages <= 0 || c->page_size <= 0 || c->n_head_kv <= 0 || c->n_seqs <= 0 || c->max_pages <= 0)
        why = "invalid argument: paged cache with an empty axis";
    else if (c->n_pages >= ((int64_t)1 << 31) || c->n_pages * c->page_size >= ((int64_t)1 << 31) ||
             (int64_t)c->max_pages * c->page_size >= ((int64_t)1 << 31) || c->n_head_kv > 65535)
        why = "invalid argument: paged cache of 2^31 cells or more, or more than 65535 heads";
    else if (c->table_stride != 0 && (c->table_stride < c->max_pages || c->table_stride >= ((int64_t)1 << 40)))
        why = "invalid argument: page table rows overlap";
    if (why) { alb_set_last_error_msg(why); return false; }
    kv.k = (uint16_t *)c->k;
    kv.v = (uint16_t *)c->v;
    kv.table = c->page_table;
    kv.table_stride = c->table_stride ? c->table_stride : c->max_pages;
    kv.n_pages = (int32_t)c->n_pages;
    kv.n_seqs = c->n_seqs;
    kv.max_pages = c->max_pages;
    kv.page_size = c->page_size;
    kv.Hkv = c->n_head_kv;
    if (c->page_stride == 0 && c->cell_stride == 0 && c->head_stride == 0) {
        kv.head_stride = c->head_dim;
        kv.cell_stride = kv.head_stride * c->n_head_kv;
        kv.page_stride = kv.cell_stride * c->page_size;
    } else {
        kv.page_stride = c->page_stride;
        kv.cell_stride = c->cell_stride;
        kv.head_stride = c->head_stride;
        Axis a[3] = {{c->page_stride, c->n_pages}, {c->cell_stride, c->page_size}, {c->head_stride, c->n_head_kv}};
        for (int i = 0; i < 2; ++i)
            for (int j = 0; j < 2 - i; ++j)
                if (a[j].stride > a[j + 1].stride) { const Axis x = a[j]; a[j] = a[j + 1]; a[j + 1] = x; }
        int64_t span = c->head_dim;
        for (const Axis & x : a) {
            if (x.count == 1 && x.stride >= 0 && x.stride % 8 == 0) continue;   // an axis of one is never stepped
            if (x.stride < span || x.stride % 8 != 0 || x.stride > ((int64_t)1 << 44) / x.count) {
                alb_set_last_error_msg("invalid argument: paged cache strides overlap, are no multiples of 8 or too large");
                return false;
            }
            span = x.stride * x.count;
        }
    }
    uint32_t s = 0;
    while (((uint64_t)1 << s) < (uint64_t)c->page_size) ++s;
    kv.div_shift = s;
    kv.div_mul = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << s) - (uint64_t)c->page_size)) / (uint64_t)c->page_size + 1);
    return true;
}

template <int D, bool BF16>
cudaError_t launch_append(const float * qkv, int64_t qkv_stride, int64_t T, int Hq, const float * qn, const float * kn,
                          float eps, const float * rope, int32_t max_pos, const int32_t * positions,
                          const int32_t * seqs, const PagedView & kv, float * q_out, int * err, cudaStream_t st) {
    const int64_t items = T * (Hq + 2 * kv.Hkv);
    return alb_launch(k_qk_norm_rope_kv_paged<D, BF16>, dim3((unsigned)((items + 7) / 8)), dim3(256), 0, st, true, qkv,
                      qkv_stride, items, Hq, qn, kn, eps, rope, max_pos, positions, seqs, kv, q_out, err);
}

template <int D, bool BF16>
cudaError_t launch_attn(const float * q, int64_t n_rows, int Hq, const PagedView & kv, const int32_t * seqs,
                        const int32_t * lengths, int32_t window, float scale, float * out, float * lse, int * err,
                        cudaStream_t st) {
    return alb_launch(k_paged_attn<D, BF16>, dim3((unsigned)n_rows, (unsigned)Hq), dim3(128), 0, st, true, q, Hq, kv,
                      seqs, lengths, window, scale, out, lse, err);
}

}  // namespace

extern "C" int alb_qk_norm_rope_kv_paged(const float * qkv, int64_t qkv_stride, int64_t T, int32_t n_head,
                                         const float * q_norm, const float * k_norm, float eps,
                                         const float * rope_table, int32_t max_pos, const int32_t * positions,
                                         const int32_t * seqs, const alb_paged_kv * kv, float * q_out, void * stream) {
    PagedView v;
    if (!paged_view(kv, v, true)) return ALB_ERR_INVALID;
    ALB_CHECK_ARG(qkv && rope_table && positions && q_out && T > 0 && max_pos > 0 && eps >= 0.0f);
    ALB_CHECK_ARG(n_head > 0 && n_head <= 65535 && T <= ((int64_t)1 << 31) / (n_head + 2 * v.Hkv));
    const int64_t dense = (int64_t)(n_head + 2 * v.Hkv) * kv->head_dim;
    ALB_CHECK_ARG(qkv_stride == 0 || (qkv_stride >= dense && qkv_stride % 4 == 0 && qkv_stride < ((int64_t)1 << 31)));
    ALB_CHECK_ARG((((uintptr_t)qkv | (uintptr_t)q_norm | (uintptr_t)k_norm | (uintptr_t)rope_table | (uintptr_t)q_out) & 15) == 0);
    int * err = device_error_ptr();
    ALB_CUDA_TRY(err ? cudaSuccess : cudaErrorMemoryAllocation);
    auto * f = kv->head_dim == 128 ? (kv->type == ALB_KV_BF16 ? launch_append<128, true> : launch_append<128, false>)
                                   : (kv->type == ALB_KV_BF16 ? launch_append<64, true> : launch_append<64, false>);
    ALB_CUDA_TRY(f(qkv, qkv_stride ? qkv_stride : dense, T, n_head, q_norm, k_norm, eps, rope_table, max_pos,
                   positions, seqs, v, q_out, err, (cudaStream_t)stream));
    return ALB_OK;
}

extern "C" size_t alb_paged_attn_workspace_bytes(const alb_paged_kv * kv, int64_t n_rows, int32_t n_head) {
    PagedView v;
    if (!paged_view(kv, v, false) || n_rows <= 0 || n_head <= 0 || n_head % v.Hkv != 0) return 0;
    return 16;
}

extern "C" int alb_paged_attn(const float * q, int64_t n_rows, int32_t n_head, const alb_paged_kv * kv,
                              const int32_t * seqs, const int32_t * lengths, int32_t window, float scale,
                              void * workspace, float * out, float * lse, void * stream) {
    PagedView v;
    if (!paged_view(kv, v, true)) return ALB_ERR_INVALID;
    ALB_CHECK_ARG(q && lengths && workspace && out && n_rows > 0 && n_rows < ((int64_t)1 << 24) && window >= 0);
    ALB_CHECK_ARG(n_head > 0 && n_head <= 65535 && n_head % v.Hkv == 0);
    ALB_CHECK_ARG(scale > 0.0f && std::isfinite(scale));
    ALB_CHECK_ARG((((uintptr_t)q | (uintptr_t)out | (uintptr_t)workspace) & 15) == 0);
    int * err = device_error_ptr();
    ALB_CUDA_TRY(err ? cudaSuccess : cudaErrorMemoryAllocation);
    auto * f = kv->head_dim == 128 ? (kv->type == ALB_KV_BF16 ? launch_attn<128, true> : launch_attn<128, false>)
                                   : (kv->type == ALB_KV_BF16 ? launch_attn<64, true> : launch_attn<64, false>);
    ALB_CUDA_TRY(f(q, n_rows, n_head, v, seqs, lengths, window, scale, out, lse, err, (cudaStream_t)stream));
    return ALB_OK;
}
