// Logits of a batch before its tokens are chosen (sm_100a): biases, penalties
// for repeated tokens, temperature, grammar masks and the greedy token in one
// pass over the rows.
//
// A row belongs to one thread-block cluster whose CTAs share the vocabulary.
// Each CTA counts its share of tokens in a table in shared memory: the row's
// history is read once, every CTA taking a part of it and adding each id into
// the table of the CTA that owns it (distributed shared memory, integer atomics,
// so the counts do not depend on their order).  Then every CTA streams its share
// of the logits once, and the row's maximum is joined in CTA 0's shared memory.
#include "alb_common.cuh"
#include "alb_internal.h"

using namespace alb;

namespace {

constexpr int LG_THREADS = 512;
constexpr int LG_MAX_CLUSTER = 16;
constexpr uint32_t LG_PROMPT = 1u << 31, LG_BIASED = 1u << 30, LG_COUNT = LG_BIASED - 1;

struct LogitsArgs {
    const float * x;
    float * y;
    int64_t n_vocab, x_stride, y_stride;
    int32_t * next;
    alb_logits_rules r;
    int64_t chunk;       // tokens per CTA, a multiple of 4
    int table;           // 1: the CTA keeps a table of counts
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

struct RowRules { float rep, freq, pres, temp; };

// The rules on one value, c its table entry, `allowed` its mask bit.
__device__ __forceinline__ float lg_value(float x, uint32_t c, bool allowed, const RowRules & k) {
    if (c & (LG_PROMPT | LG_COUNT)) {
        x = x > 0.0f ? __fdiv_rn(x, k.rep) : __fmul_rn(x, k.rep);
        const uint32_t n = c & LG_COUNT;
        if (n) x = __fsub_rn(__fsub_rn(x, __fmul_rn(k.freq, (float)n)), k.pres);
    }
    if (k.temp > 0.0f) x = __fdiv_rn(x, k.temp);
    return allowed ? x : -INFINITY;
}

// (value, index) as one ordered number: larger values first, then lower
// indices; 0 for -INFINITY and NaN, which are never chosen.
__device__ __forceinline__ unsigned long long lg_key(float v, int64_t i) {
    if (!(v > -INFINITY)) return 0ull;
    uint32_t u = __float_as_uint(v == 0.0f ? 0.0f : v);
    u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((unsigned long long)u << 32) | (uint32_t)(0x7FFFFFFF - (int32_t)i);
}

__global__ void __launch_bounds__(LG_THREADS)
k_logits(const __grid_constant__ LogitsArgs a) {
    extern __shared__ __align__(16) uint32_t table[];   // [chunk]
    __shared__ unsigned long long red[LG_THREADS / 32], joined[LG_MAX_CLUSTER];
    uint32_t rank, size;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
    const int64_t row = blockIdx.x / size;
    const int tid = threadIdx.x, lane = tid & 31;
    alb_pdl_wait();
    const alb_logits_rules & r = a.r;
    int32_t len = r.history_len ? r.history_len[row] : (int32_t)r.history_stride;
    if (len < 0) { alb_pdl_trigger(); return; }   // a padding row: all CTAs of its cluster leave here
    bool bad = false;
    if (r.history && len > r.history_stride) { len = (int32_t)r.history_stride; bad = true; }
    const float * x = a.x + row * a.x_stride;
    float * y = a.y + row * a.y_stride;
    // tokens are dealt out in groups of four that start on 16-byte boundaries
    // of x: group g holds tokens 4 g - shift .. 4 g - shift + 3
    const int64_t shift = (int64_t)(((uintptr_t)x >> 2) & 3);
    const int64_t i0 = rank * a.chunk - shift;   // first token of this CTA's share
    if (a.table) {
        for (int64_t j = tid; j < a.chunk / 4; j += LG_THREADS) reinterpret_cast<uint4 *>(table)[j] = make_uint4(0, 0, 0, 0);
        if (r.bias_ids) {
            // the last entry of an id counts: the table first takes the largest
            // entry number per id, whose thread then leaves x + bias in y and a
            // mark; CTAs look only at ids of their own share
            int32_t b0 = r.bias_offsets[row], b1 = r.bias_offsets[row + 1];
            if (b0 < 0 || b1 > r.n_bias) { bad = true; b0 = max(b0, 0); b1 = min(b1, r.n_bias); }
            __syncthreads();
            for (int32_t e = b0 + tid; e < b1; e += LG_THREADS) {
                const int32_t id = r.bias_ids[e];
                if (id >= a.n_vocab) { bad = true; continue; }
                const int64_t j = id - i0;
                if (id >= 0 && j >= 0 && j < a.chunk) atomicMax(table + j, (uint32_t)(e - b0) + 1u);
            }
            __syncthreads();
            for (int32_t e = b0 + tid; e < b1; e += LG_THREADS) {
                const int32_t id = r.bias_ids[e];
                const int64_t j = id - i0;
                if (id < 0 || id >= a.n_vocab || j < 0 || j >= a.chunk || table[j] != (uint32_t)(e - b0) + 1u) continue;
                y[id] = __fadd_rn(x[id], r.bias_values[e]);
                table[j] = LG_BIASED;   // (entry numbers stay below the mark: no other entry matches it)
            }
        }
        lg_cluster_sync();   // every table is ready for the others' ids
        if (r.history) {
            const int32_t start = r.last_n > 0 && len > r.last_n ? len - r.last_n : 0;
            const int32_t prompt = r.prompt_len ? r.prompt_len[row] : 0;
            const int32_t * h = r.history + row * r.history_stride;
            const uint32_t base = alb_smem_addr(table);
            for (int32_t e = start + (int32_t)rank * LG_THREADS + tid; e < len; e += (int32_t)size * LG_THREADS) {
                const int32_t id = h[e];
                if (id < 0) continue;
                if (id >= a.n_vocab) { bad = true; continue; }
                const uint32_t at = (uint32_t)(id + shift), owner = at / (uint32_t)a.chunk;
                uint32_t dst;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                             : "=r"(dst) : "r"(base + 4u * (at - owner * (uint32_t)a.chunk)), "r"(owner));
                if (e < prompt) asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" :: "r"(dst), "r"(LG_PROMPT) : "memory");
                else            asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" :: "r"(dst), "r"(1u) : "memory");
            }
        }
        lg_cluster_sync();   // every id is counted
    }
    const RowRules k = {r.repetition ? r.repetition[row] : 1.0f, r.frequency ? r.frequency[row] : 0.0f,
                        r.presence ? r.presence[row] : 0.0f, r.temperature ? r.temperature[row] : 0.0f};
    const uint32_t * allow = nullptr;
    if (r.allow) {
        const int64_t m = r.allow_row ? r.allow_row[row] : row;
        if (m >= r.n_allow) bad = true;
        else if (m >= 0) allow = r.allow + m * r.allow_stride;
    }
    unsigned long long best = 0;
    for (int64_t j = 4 * tid; j < a.chunk; j += 4 * LG_THREADS) {
        const int64_t i = i0 + j;
        if (i >= a.n_vocab) break;
        uint4 c = make_uint4(0, 0, 0, 0);
        if (a.table) c = *reinterpret_cast<const uint4 *>(table + j);
        const uint32_t cs[4] = {c.x, c.y, c.z, c.w};
        float v[4];
        const bool whole = i >= 0 && i + 4 <= a.n_vocab;
        if (whole) *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(x + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (i + e < 0 || i + e >= a.n_vocab) continue;
            if (!whole) v[e] = x[i + e];
            if (cs[e] & LG_BIASED) v[e] = y[i + e];
            bool allowed = true;
            if (allow) allowed = (allow[(i + e) >> 5] >> ((i + e) & 31)) & 1u;
            v[e] = lg_value(v[e], cs[e], allowed, k);
            const unsigned long long key = lg_key(v[e], i + e);
            best = key > best ? key : best;
        }
        if (whole && a.vec_out) {
            *reinterpret_cast<float4 *>(y + i) = *reinterpret_cast<float4 *>(v);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e >= 0 && i + e < a.n_vocab) y[i + e] = v[e];
        }
    }
    if (bad) atomicExch(a.err, ALB_DEVERR_BAD_INDEX);
    if (a.next) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
            best = other > best ? other : best;
        }
        if (lane == 0) red[tid >> 5] = best;
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < LG_THREADS / 32; ++w) best = red[w] > best ? red[w] : best;
            asm volatile("st.shared::cluster.u64 [%0], %1;" :: "r"(lg_remote(&joined[rank], 0)), "l"(best) : "memory");
        }
        lg_cluster_sync();
        if (rank == 0 && tid == 0) {
            for (uint32_t w = 0; w < size; ++w) best = joined[w] > best ? joined[w] : best;
            a.next[row] = best ? 0x7FFFFFFF - (int32_t)(uint32_t)best : -1;
        }
    }
    alb_pdl_trigger();
}

cudaError_t launch_logits(const LogitsArgs & a, int64_t rows, int cluster, cudaStream_t st) {
    const size_t smem = a.table ? (size_t)a.chunk * 4 : 0;
    cudaError_t e = ensure_smem(k_logits, smem);
    if (e == cudaSuccess && cluster > 8) e = cudaFuncSetAttribute(k_logits, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * cluster));
    cfg.blockDim = dim3(LG_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, k_logits, a);
}

}  // namespace

extern "C" int alb_logits_process(const float * logits, int64_t rows, int64_t n_vocab, int64_t stride,
                                  const alb_logits_rules * rules, float * out, int64_t out_stride,
                                  int32_t * next_token, void * stream) {
    ALB_CHECK_ARG(logits && rules && out && rows > 0 && rows < ((int64_t)1 << 24));
    ALB_CHECK_ARG(n_vocab > 0 && n_vocab < ((int64_t)1 << 31) - 64);
    const alb_logits_rules & r = *rules;
    const int64_t xs = stride ? stride : n_vocab, ys = out_stride ? out_stride : n_vocab;
    ALB_CHECK_ARG(xs >= n_vocab && ys >= n_vocab && xs < ((int64_t)1 << 36) && ys < ((int64_t)1 << 36));
    ALB_CHECK_ARG((((uintptr_t)logits | (uintptr_t)out) & 3) == 0);
    // in place means the same rows; any other overlap would change rows that are still to be read
    const uintptr_t x0 = (uintptr_t)logits, x1 = x0 + 4 * (uintptr_t)((rows - 1) * xs + n_vocab);
    const uintptr_t y0 = (uintptr_t)out, y1 = y0 + 4 * (uintptr_t)((rows - 1) * ys + n_vocab);
    ALB_CHECK_ARG((logits == out && (xs == ys || rows == 1)) || x1 <= y0 || y1 <= x0);
    ALB_CHECK_ARG(!r.history || (r.history_stride > 0 && r.history_stride < (1 << 30)));
    ALB_CHECK_ARG(r.last_n >= 0);
    ALB_CHECK_ARG(!r.bias_ids || (r.bias_values && r.bias_offsets && r.n_bias >= 0 && r.n_bias < (1 << 30)));
    ALB_CHECK_ARG(!r.allow || (r.n_allow > 0 && (r.allow_stride == 0 || r.allow_stride >= (n_vocab + 31) / 32)));
    LogitsArgs a = {};
    a.x = logits; a.y = out; a.n_vocab = n_vocab; a.x_stride = xs; a.y_stride = ys; a.next = next_token; a.r = r;
    if (!r.repetition && !r.frequency && !r.presence) a.r.history = nullptr;   // nothing asks for the counts
    if (!a.r.history) a.r.history_stride = 0;
    if (r.allow && !r.allow_stride) a.r.allow_stride = (n_vocab + 31) / 32;
    a.table = a.r.history || r.bias_ids;
    ALB_CHECK_ARG(!a.table || n_vocab <= (1 << 19));
    // every row starts on the same 16-byte phase in x and y (or all by four bytes)
    a.vec_out = (((uintptr_t)logits ^ (uintptr_t)out) & 15) == 0 && (rows == 1 || ((xs ^ ys) & 3) == 0);
    int cluster = 8;
    if (a.table && n_vocab > 8 * 25600) cluster = 16;
    a.chunk = (((n_vocab + 3 + cluster - 1) / cluster) + 3) & ~(int64_t)3;   // + 3: the first group may start before the row
    a.err = device_error_ptr();
    ALB_CUDA_TRY(a.err ? cudaSuccess : cudaErrorMemoryAllocation);
    ALB_CUDA_TRY(launch_logits(a, rows, cluster, (cudaStream_t)stream));
    return ALB_OK;
}
