// Logits of a batch before its tokens are chosen (sm_100a): biases, penalties
// for repeated tokens, temperature, grammar masks and the greedy token in one
// pass over the rows.
//
// A row belongs to one thread-block cluster whose CTAs share the vocabulary,
// granules of 128 tokens dealt out in turn (frequent tokens have neighbouring
// ids).  Each CTA counts its tokens in a table in shared memory: it reads the
// row's whole history and adds up the ids it owns, with integer atomics, so the
// counts do not depend on their order.  Each counted or biased entry is then
// replaced, once, by its token's value with bias and penalties.  What is left
// for the stream over the logits is the same for every token: the table's value
// where there is one, temperature, mask, maximum; the row's maximum is joined in
// CTA 0's shared memory.
#include "alb_common.cuh"
#include "alb_internal.h"

using namespace alb;

namespace {

constexpr int LG_THREADS = 512;
constexpr int LG_BATCH = 5;              // 16-byte loads of logits in flight per thread
constexpr int LG_MAX_CLUSTER = 16;
constexpr int LG_LIST = 1024;            // distinct ids of a CTA that it remembers (more: it reads the history again)

// A table entry is a token's value once that is known, and before that a NaN
// that no value is stored as: LG_FREE plus the token's count in the output, and
// two marks (the id is in the prompt; its logit with bias waits in y).
// LG_TAKEN: a thread is working on its value.
constexpr uint32_t LG_FREE = 0xFFC00000u, LG_PROMPT = 1u << 21, LG_BIASED = 1u << 20, LG_TAKEN = 0xFFFFFFFFu;
constexpr int64_t LG_MAX_HISTORY = LG_BIASED - 1;   // counts stay below the marks

struct LogitsArgs {
    const float * x;
    float * y;
    int64_t n_vocab, x_stride, y_stride;
    int32_t * next;
    alb_logits_rules r;
    int32_t granules;    // granules of 128 tokens per CTA
    int32_t log_cluster;
    int vec_out;         // 1: y's rows have the alignment of x's
    int * err;
};

__device__ __forceinline__ void lg_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t lg_remote(const void * local, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(alb_smem_addr(local)), "r"(rank));
    return a;
}
__device__ __forceinline__ float4 lg_load(const float * p) {   // (not .nc: y may be x)
    float4 v;
    asm volatile("ld.global.L1::no_allocate.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p) : "memory");
    return v;
}

// x / t rounded to nearest, for r = 1 / t rounded to nearest and 2^-100 < |x| <
// 2^100, 2^-20 < t < 2^20 (nothing under- or overflows): the quotient is brought
// within one step by the first correction, and by Markstein's theorem ("Computation
// of elementary functions on the IBM RISC System/6000 processor", 1990) the second
// one rounds it as the exact quotient.  (t's significand all ones, which the
// theorem leaves out for r itself, does no harm: r is rounded from the exact 1 / t.)
__device__ __forceinline__ float lg_divide(float x, float t, float r) {
    float q = __fmul_rn(x, r);
    q = __fmaf_rn(__fmaf_rn(-q, t, x), r, q);
    return __fmaf_rn(__fmaf_rn(-q, t, x), r, q);
}

// TABLE: whether ids are counted or biased at all.
template <bool TABLE>
__global__ void __launch_bounds__(LG_THREADS, 1024 / LG_THREADS)
k_logits(const __grid_constant__ LogitsArgs a) {
    extern __shared__ __align__(16) uint32_t table[];   // [granules * 128]
    __shared__ float red_v[LG_THREADS / 32];
    __shared__ int32_t red_i[LG_THREADS / 32];
    __shared__ int2 joined[LG_MAX_CLUSTER];
    __shared__ int32_t list[TABLE ? LG_LIST : 1], n_list;
    const uint32_t rank = blockIdx.x & ((1u << a.log_cluster) - 1u);   // (clusters are runs of the one-dimensional grid)
    const int64_t row = blockIdx.x >> a.log_cluster;
    const int tid = threadIdx.x, lane = tid & 31;
    const int32_t groups = a.granules * 32;
    if (TABLE) {
        for (int32_t j = tid; j < groups; j += LG_THREADS)
            reinterpret_cast<uint4 *>(table)[j] = make_uint4(LG_FREE, LG_FREE, LG_FREE, LG_FREE);
        if (tid == 0) n_list = 0;
    }
    alb_pdl_wait();
    alb_pdl_trigger();
    const alb_logits_rules & r = a.r;
    int32_t len = r.history_len ? r.history_len[row] : (int32_t)r.history_stride;
    if (len < 0) return;   // a padding row: all CTAs of its cluster leave here
    bool bad = false;
    if (r.history && len > r.history_stride) { len = (int32_t)r.history_stride; bad = true; }
    const float * x = a.x + row * a.x_stride;
    float * y = a.y + row * a.y_stride;
    const int32_t n_vocab = (int32_t)a.n_vocab;
    // token i is place i + shift, so that groups of four places start on 16-byte boundaries of x
    const int32_t shift = (int32_t)(((uintptr_t)x >> 2) & 3);
    // group q of this CTA: the first of its four tokens (may lie outside [0, n_vocab))
    auto token_of = [&](int32_t q) {
        return (int32_t)(((((uint32_t)q >> 5) << a.log_cluster) + rank) << 7) + ((q & 31) << 2) - shift;
    };
    // whether this CTA owns token id, and its table entry
    auto owned = [&](int32_t id, uint32_t & j) {
        const uint32_t at = (uint32_t)(id + shift), gr = at >> 7;
        j = ((gr >> a.log_cluster) << 7) | (at & 127u);
        return (gr & ((1u << a.log_cluster) - 1u)) == rank;
    };
    auto whole = [&](int32_t i) { return i >= 0 && i <= n_vocab - 4; };
    float4 v[LG_BATCH];
    auto load = [&](int32_t q0) {
#pragma unroll
        for (int u = 0; u < LG_BATCH; ++u) {
            const int32_t q = q0 + u * LG_THREADS, i = token_of(q);
            if (q < groups && whole(i)) v[u] = lg_load(x + i);
        }
    };
    load(tid);   // the first batch comes while the ids are counted

    if (TABLE) {
        const float rep = r.repetition ? r.repetition[row] : 1.0f, freq = r.frequency ? r.frequency[row] : 0.0f;
        const float pres = r.presence ? r.presence[row] : 0.0f;
        __syncthreads();   // the table is free
        int32_t b0 = 0, b1 = 0;
        if (r.bias_ids) {
            // the last entry of an id counts: blocks of entries from the back, within a block the
            // largest place wins the table entry; its thread leaves x + bias in y and a mark that
            // keeps earlier entries away
            b0 = r.bias_offsets[row];
            b1 = r.bias_offsets[row + 1];
            if (b0 < 0 || b1 > r.n_bias) { bad = true; b0 = max(b0, 0); b1 = min(b1, r.n_bias); }
            for (int32_t end = b1; end > b0; end -= LG_THREADS) {
                const int32_t e = end - 1 - tid;
                const uint32_t place = LG_FREE + LG_THREADS - tid;
                uint32_t j = 0;
                int32_t id = -1;
                if (e >= b0) {
                    id = r.bias_ids[e];
                    if (id >= n_vocab) { bad = true; id = -1; }
                    if (id >= 0 && (!owned(id, j) || (table[j] & LG_BIASED))) id = -1;
                }
                __syncthreads();   // marks are read before places go in
                if (id >= 0) atomicMax(table + j, place);
                __syncthreads();
                const bool won = id >= 0 && table[j] == place;
                __syncthreads();
                if (won) {
                    y[id] = __fadd_rn(x[id], r.bias_values[e]);
                    table[j] = LG_FREE | LG_BIASED;
                }
                __syncthreads();
            }
        }
        const int32_t start = r.last_n > 0 && len > r.last_n ? len - r.last_n : 0;
        const int32_t prompt = r.history && r.prompt_len ? r.prompt_len[row] : 0;
        const int32_t * h = r.history + row * r.history_stride;
        // every id of the counted history: f(position, id)
        auto each = [&](auto && f) {
            if (!r.history) return;
            for (int32_t e = start + tid; e < len; e += 4 * LG_THREADS) {
                int32_t id[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) id[u] = e + u * LG_THREADS < len ? h[e + u * LG_THREADS] : -1;
#pragma unroll
                for (int u = 0; u < 4; ++u) f(e + u * LG_THREADS, id[u]);
            }
        };
        each([&](int32_t e, int32_t id) {
            uint32_t j;
            if (id >= n_vocab) bad = true;
            if (id < 0 || id >= n_vocab || !owned(id, j)) return;
            if ((e < prompt ? atomicOr(table + j, LG_PROMPT) : atomicAdd(table + j, 1u)) == LG_FREE) {
                const int at = atomicAdd(&n_list, 1);   // the first place of this id
                if (at < LG_LIST) list[at] = id;
            }
        });
        __syncthreads();   // every id is counted
        auto settle = [&](int32_t id) {
            uint32_t j;
            if (id < 0 || id >= n_vocab || !owned(id, j)) return;
            const uint32_t c = *reinterpret_cast<volatile uint32_t *>(table + j);
            // an entry whose value is known, or taken by the thread of the same id's other place, is left
            if (c <= LG_FREE || c == LG_TAKEN || atomicCAS(table + j, c, LG_TAKEN) != c) return;
            float f = (c & LG_BIASED) ? y[id] : x[id];
            const uint32_t n = c & (LG_BIASED - 1u);
            if (n || (c & LG_PROMPT)) f = f > 0.0f ? __fdiv_rn(f, rep) : __fmul_rn(f, rep);
            if (n) f = __fsub_rn(__fsub_rn(f, __fmul_rn(freq, (float)n)), pres);
            table[j] = f == f ? __float_as_uint(f) : 0x7FC00000u;
        };
        if (n_list <= LG_LIST)
            for (int32_t e = tid; e < n_list; e += LG_THREADS) settle(list[e]);
        else
            each([&](int32_t, int32_t id) { settle(id); });
        for (int32_t e = b0 + tid; e < b1; e += LG_THREADS) settle(r.bias_ids[e]);
    }
    const float temp = r.temperature ? r.temperature[row] : 0.0f;
    const bool plain_temp = temp > 0x1p-20f && temp < 0x1p20f;
    const float inv = plain_temp ? __frcp_rn(temp) : 0.0f;
    const uint32_t * allow = nullptr;
    if (r.allow) {
        const int64_t m = r.allow_row ? r.allow_row[row] : row;
        if (m >= r.n_allow) bad = true;
        else if (m >= 0) allow = r.allow + m * r.allow_stride;
    }
    if (TABLE) __syncthreads();   // every value is in place
    float best = -INFINITY;
    int32_t best_i = -1;
    for (int32_t q0 = tid; q0 < groups;) {
#pragma unroll
        for (int u = 0; u < LG_BATCH; ++u) {
            const int32_t q = q0 + u * LG_THREADS, i = token_of(q);
            if (q >= groups || i >= n_vocab) continue;
            const bool all = whole(i);
            float f[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
            if (!all) {
#pragma unroll
                for (int e = 0; e < 4; ++e) f[e] = i + e >= 0 && i + e < n_vocab ? x[i + e] : -INFINITY;
            }
            if (TABLE) {
                const uint4 c = reinterpret_cast<const uint4 *>(table)[q];
                f[0] = c.x == LG_FREE ? f[0] : __uint_as_float(c.x);
                f[1] = c.y == LG_FREE ? f[1] : __uint_as_float(c.y);
                f[2] = c.z == LG_FREE ? f[2] : __uint_as_float(c.z);
                f[3] = c.w == LG_FREE ? f[3] : __uint_as_float(c.w);
            }
            if (temp > 0.0f) {
                const float lo = fminf(fminf(fabsf(f[0]), fabsf(f[1])), fminf(fabsf(f[2]), fabsf(f[3])));
                const float hi = fmaxf(fmaxf(fabsf(f[0]), fabsf(f[1])), fmaxf(fabsf(f[2]), fabsf(f[3])));
                if (plain_temp && lo > 0x1p-100f && hi < 0x1p100f) {   // (a NaN among them stays NaN either way)
#pragma unroll
                    for (int e = 0; e < 4; ++e) f[e] = lg_divide(f[e], temp, inv);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) f[e] = __fdiv_rn(f[e], temp);
                }
            }
            if (allow) {
                const int32_t w0 = max(i, 0) >> 5, w1 = min(i + 3, n_vocab - 1) >> 5;
                const uint32_t lo = allow[w0], hi = allow[w1];
                // bit e of `bits`: token i + e (the bits of tokens outside the row are not used)
                const uint32_t bits = i >= 0 ? __funnelshift_r(lo, hi, i & 31) : lo << -i;
#pragma unroll
                for (int e = 0; e < 4; ++e) f[e] = (bits >> e) & 1u ? f[e] : -INFINITY;
            }
            const float top = fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3]));   // (fmaxf passes over NaN)
            if (top > best) {   // a later group wins only if it is larger: the lowest index stays
                best = top;
                best_i = i + (f[0] == top ? 0 : f[1] == top ? 1 : f[2] == top ? 2 : 3);
            }
            if (all && a.vec_out) {
                *reinterpret_cast<float4 *>(y + i) = make_float4(f[0], f[1], f[2], f[3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (i + e >= 0 && i + e < n_vocab) y[i + e] = f[e];
            }
        }
        q0 += LG_BATCH * LG_THREADS;
        load(q0);
    }
    if (bad) atomicExch(a.err, ALB_DEVERR_BAD_INDEX);
    if (a.next) {
        // largest value, then lowest index (-1, from -INFINITY and NaN alone, never beats a value)
        auto take = [&](float bv, int32_t bi) {
            if (bv > best || (bv == best && (uint32_t)bi < (uint32_t)best_i)) { best = bv; best_i = bi; }
        };
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            take(__shfl_xor_sync(0xffffffffu, best, o), __shfl_xor_sync(0xffffffffu, best_i, o));
        if (lane == 0) { red_v[tid >> 5] = best; red_i[tid >> 5] = best_i; }
        __syncthreads();
        if (tid < 32) {
            best = tid < LG_THREADS / 32 ? red_v[tid] : -INFINITY;
            best_i = tid < LG_THREADS / 32 ? red_i[tid] : -1;
#pragma unroll
            for (int o = 8; o > 0; o >>= 1)
                take(__shfl_xor_sync(0xffffffffu, best, o), __shfl_xor_sync(0xffffffffu, best_i, o));
            if (tid == 0)
                asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};"
                             :: "r"(lg_remote(&joined[rank], 0)), "r"(__float_as_uint(best)), "r"(best_i) : "memory");
        }
        lg_cluster_sync();
        if (rank == 0 && tid == 0) {
            for (int w = 0; w < 1 << a.log_cluster; ++w) take(__uint_as_float((uint32_t)joined[w].x), joined[w].y);
            a.next[row] = best_i;
        }
    }
}

template <bool TABLE>
cudaError_t launch_logits(const LogitsArgs & a, int64_t rows, cudaStream_t st) {
    const size_t smem = TABLE ? (size_t)a.granules * 512 : 0;
    const unsigned cluster = 1u << a.log_cluster;
    cudaError_t e = ensure_smem(k_logits<TABLE>, smem);
    if (e == cudaSuccess && cluster > 8)
        e = cudaFuncSetAttribute(k_logits<TABLE>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * cluster));
    cfg.blockDim = dim3(LG_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, k_logits<TABLE>, a);
}

}  // namespace

extern "C" int alb_logits_process(const float * logits, int64_t rows, int64_t n_vocab, int64_t stride,
                                  const alb_logits_rules * rules, float * out, int64_t out_stride,
                                  int32_t * next_token, void * stream) {
    ALB_CHECK_ARG(logits && rules && out && rows > 0 && rows < ((int64_t)1 << 24));
    ALB_CHECK_ARG(n_vocab > 0 && n_vocab <= (1 << 30));
    const alb_logits_rules & r = *rules;
    const int64_t xs = stride ? stride : n_vocab, ys = out_stride ? out_stride : n_vocab;
    ALB_CHECK_ARG(xs >= n_vocab && ys >= n_vocab && xs < ((int64_t)1 << 36) && ys < ((int64_t)1 << 36));
    ALB_CHECK_ARG((((uintptr_t)logits | (uintptr_t)out) & 3) == 0);
    // in place means the same rows; any other overlap would change rows that are still to be read
    const uintptr_t x0 = (uintptr_t)logits, x1 = x0 + 4 * (uintptr_t)((rows - 1) * xs + n_vocab);
    const uintptr_t y0 = (uintptr_t)out, y1 = y0 + 4 * (uintptr_t)((rows - 1) * ys + n_vocab);
    ALB_CHECK_ARG((logits == out && (xs == ys || rows == 1)) || x1 <= y0 || y1 <= x0);
    ALB_CHECK_ARG(!r.history || (r.history_stride > 0 && r.history_stride <= LG_MAX_HISTORY));
    ALB_CHECK_ARG(r.last_n >= 0);
    ALB_CHECK_ARG(!r.bias_ids || (r.bias_values && r.bias_offsets && r.n_bias >= 0 && r.n_bias < (1 << 30)));
    ALB_CHECK_ARG(!r.allow || (r.n_allow > 0 && (r.allow_stride == 0 || r.allow_stride >= (n_vocab + 31) / 32)));
    LogitsArgs a = {};
    a.x = logits; a.y = out; a.n_vocab = n_vocab; a.x_stride = xs; a.y_stride = ys; a.next = next_token; a.r = r;
    if (!r.repetition && !r.frequency && !r.presence) a.r.history = nullptr;   // nothing asks for the counts
    if (!a.r.history) a.r.history_stride = 0;
    if (r.allow && !r.allow_stride) a.r.allow_stride = (n_vocab + 31) / 32;
    const bool table = a.r.history || r.bias_ids;
    ALB_CHECK_ARG(!table || n_vocab <= (1 << 19));
    // every row starts on the same 16-byte phase in x and y (or all by four bytes)
    a.vec_out = (((uintptr_t)logits ^ (uintptr_t)out) & 15) == 0 && (rows == 1 || ((xs ^ ys) & 3) == 0);
    const int64_t granules = (n_vocab + 3 + 127) / 128;   // + 3: the first group may start before the row
    a.log_cluster = rows <= 8 || (table && granules * 512 > 8 * 102400) ? 4 : 3;
    a.granules = (int32_t)((granules + (1 << a.log_cluster) - 1) >> a.log_cluster);
    a.err = device_error_ptr();
    ALB_CUDA_TRY(a.err ? cudaSuccess : cudaErrorMemoryAllocation);
    ALB_CUDA_TRY((table ? launch_logits<true> : launch_logits<false>)(a, rows, (cudaStream_t)stream));
    return ALB_OK;
}
