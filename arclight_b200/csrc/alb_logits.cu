// Logits of a batch before its tokens are chosen (sm_100a): biases, penalties
// for repeated tokens, temperature, grammar masks and the greedy token in one
// pass over the rows.
//
// A row belongs to one thread-block cluster whose CTAs share the vocabulary,
// granules of 128 tokens dealt out in turn (frequent tokens have neighbouring
// ids).  A CTA sends its share of the logits on the way to the L2 cache, then
// reads the row's whole history and counts the ids it owns in a table in shared
// memory (integer atomics, so the counts do not depend on their order); whoever
// counts an id first puts it on a list.  The value of each listed id is settled,
// bias and penalties applied, and what is left for the one pass over the logits
// is the same for every token: the settled value where there is one, temperature,
// mask, maximum.  The CTAs' maxima go to CTA 0's shared memory.
//
// Bound by instruction issue and the chain of dependent steps, not by HBM: 256
// rows of 151936 with histories to 4096 and masks take 83 us (314 MB, 3.8 TB/s).
// A warp issues about 1700 instructions there: 520 for copy and maximum of its nine
// groups of four tokens a lane, 190 for the temperature, 240 for the mask, 330 to
// look into the table, and 110 for each id that its lanes read, four on average.
// 48 rows with biases and masks take 20 us, 64 rows of 32003 with histories to 8192
// 13 us, one row 4.8 us.  Other shapes that were measured on the first of
// these: ids counted across the cluster in distributed shared memory 113 us
// (frequent ids queue up at their owner), the share brought to shared memory by
// bulk copies 124 us (room for two CTAs), slots by a bit map's running count 97 us
// (the history read twice), clusters that stay and take rows in turn 108 us.
#include <atomic>

#include "alb_common.cuh"
#include "alb_internal.h"

using namespace alb;

namespace {

constexpr int LG_THREADS = 512;
constexpr int LG_WARPS = LG_THREADS / 32;
constexpr int LG_BATCH = 3;              // 16-byte loads of logits in flight per thread
constexpr int LG_IDS = 4;                // loads of ids in flight per thread
constexpr int LG_GRANULE = 128;          // tokens dealt out together: a group of four per lane of a warp
constexpr int LG_MAX_CLUSTER = 16;
constexpr int LG_LIST = 2048;            // ids of a CTA whose settled values it holds

// A table entry: how often the id is in the counted output, and two marks (the
// id is in the prompt; its logit with bias waits in y), until the id is settled:
// then 1 + its place on the list.  16 bits where the host knows that no count can
// reach the marks.
template <typename T> struct Entry {
    static constexpr uint32_t PROMPT = 1u << (8 * sizeof(T) - 1), BIASED = PROMPT >> 1, COUNT = BIASED - 1;
};

constexpr size_t LG_STATIC = 16384;                 // bound of the kernel's static shared memory

struct LogitsArgs {
    const float * x;
    float * y;
    int64_t n_vocab, x_stride, y_stride;
    int32_t * next;
    alb_logits_rules r;
    int32_t granules;    // granules per CTA
    int32_t log_cluster;
    int vec_out;         // 1: y's rows have the alignment of x's
    int * err;
};

// (relaxed: all that lies before it is the barrier's own initialisation, which has its fence)
__device__ __forceinline__ void lg_cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void lg_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t lg_remote(const void * local, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(alb_smem_addr(local)), "r"(rank));
    return a;
}
// 8 bytes into another CTA's shared memory, counted on that CTA's barrier.
__device__ __forceinline__ void lg_send(uint32_t dst, uint32_t bar, uint32_t lo, uint32_t hi) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];"
                 :: "r"(dst), "r"(lo), "r"(hi), "r"(bar) : "memory");
}
// An entry's count or marks; gives the entry before.
template <typename T> __device__ __forceinline__ uint32_t lg_add(T * table, uint32_t j, uint32_t v) {
    if (sizeof(T) == 4) return atomicAdd(reinterpret_cast<uint32_t *>(table) + j, v);
    const uint32_t s = 16 * (j & 1);
    return (atomicAdd(reinterpret_cast<uint32_t *>(table) + (j >> 1), v << s) >> s) & 0xFFFFu;
}
template <typename T> __device__ __forceinline__ uint32_t lg_or(T * table, uint32_t j, uint32_t v) {
    if (sizeof(T) == 4) return atomicOr(reinterpret_cast<uint32_t *>(table) + j, v);
    const uint32_t s = 16 * (j & 1);
    return (atomicOr(reinterpret_cast<uint32_t *>(table) + (j >> 1), v << s) >> s) & 0xFFFFu;
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
// one rounds it as the exact quotient.
// (Two quotients at a time.)
__device__ __forceinline__ uint64_t lg_pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void lg_divide2(float & a, float & b, uint64_t minus_t, uint64_t r) {
    const uint64_t x = lg_pair(a, b);
    uint64_t q, e;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(q) : "l"(x), "l"(r));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(e) : "l"(q), "l"(minus_t), "l"(x));
        asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(q) : "l"(e), "l"(r), "l"(q));
    }
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(q));
}

template <typename T> __device__ __forceinline__ void lg_max(T * table, uint32_t j, uint32_t v) {
    if (sizeof(T) == 4) { atomicMax(reinterpret_cast<uint32_t *>(table) + j, v); return; }
    unsigned short * p = reinterpret_cast<unsigned short *>(table) + j;
    unsigned short old = *reinterpret_cast<volatile unsigned short *>(p);
    while (old < v) {   // ends: another thread's success only raises the entry, at most LG_THREADS times
        const unsigned short was = atomicCAS(p, old, (unsigned short)v);
        if (was == old) break;
        old = was;
    }
}
// Four entries from j (a multiple of 4); whether any is set.
__device__ __forceinline__ bool lg_entries(const uint16_t * table, uint32_t j, uint32_t (&c)[4]) {
    const uint2 v = *reinterpret_cast<const uint2 *>(table + j);
    c[0] = v.x & 0xFFFFu; c[1] = v.x >> 16; c[2] = v.y & 0xFFFFu; c[3] = v.y >> 16;
    return (v.x | v.y) != 0u;
}
__device__ __forceinline__ bool lg_entries(const uint32_t * table, uint32_t j, uint32_t (&c)[4]) {
    const uint4 v = *reinterpret_cast<const uint4 *>(table + j);
    c[0] = v.x; c[1] = v.y; c[2] = v.z; c[3] = v.w;
    return (v.x | v.y | v.z | v.w) != 0u;
}
// Floats as unsigned numbers of the same order (-0 as 0).
__device__ __forceinline__ uint32_t lg_order(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

struct RowRules { float rep, freq, pres; };
template <typename T> __device__ __forceinline__ float lg_penalty(float f, uint32_t c, const RowRules & k) {
    const uint32_t n = c & Entry<T>::COUNT;
    if (c & (Entry<T>::COUNT | Entry<T>::PROMPT)) f = f > 0.0f ? __fdiv_rn(f, k.rep) : __fmul_rn(f, k.rep);
    if (n) f = __fsub_rn(__fsub_rn(f, __fmul_rn(k.freq, (float)n)), k.pres);
    return f;
}

// The same, out of line: the pass over the logits calls it only when the list was too short.
template <typename T> __device__ __noinline__ float lg_penalty_called(float f, uint32_t c, float rep, float freq, float pres) {
    return lg_penalty<T>(f, c, RowRules{rep, freq, pres});
}

// T: the table's entries; TABLE: whether ids are counted or biased at all; PER_SM:
// CTAs an SM, 2 (64 registers a thread) or 3 (40, some spilled).
template <typename T, bool TABLE, int PER_SM>
__global__ void __launch_bounds__(LG_THREADS, PER_SM)
k_logits(const __grid_constant__ LogitsArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    T * table = reinterpret_cast<T *>(smem);                            // [granules * 128]
    uint32_t * mask = reinterpret_cast<uint32_t *>(smem + (TABLE ? a.granules * (LG_GRANULE * (int)sizeof(T)) : 0));   // [granules * 4]
    __shared__ uint32_t red_v[LG_WARPS], red_i[LG_WARPS];
    __shared__ __align__(8) uint2 joined[LG_MAX_CLUSTER];
    __shared__ __align__(8) uint64_t joined_bar;
    __shared__ uint16_t list[TABLE ? LG_LIST : 1];
    __shared__ float settled[TABLE ? LG_LIST + 1 : 1];   // [0]: no value
    __shared__ uint32_t n_list;
    const uint32_t rank = blockIdx.x & ((1u << a.log_cluster) - 1u);   // (clusters are runs of the one-dimensional grid)
    const int64_t row = blockIdx.x >> a.log_cluster;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const alb_logits_rules & r = a.r;
    const float * x = a.x + row * a.x_stride;
    float * y = a.y + row * a.y_stride;
    const int32_t n_vocab = (int32_t)a.n_vocab;
    // token i is place i + shift, so that groups of four places start on 16-byte boundaries of x
    const int32_t shift = (int32_t)(((uintptr_t)x >> 2) & 3);
    // the token at place j of this CTA's share (it may lie outside [0, n_vocab))
    auto token_of = [&](uint32_t j) {
        return (int32_t)((((j / LG_GRANULE) << a.log_cluster) + rank) * LG_GRANULE + j % LG_GRANULE) - shift;
    };
    // whether this CTA owns token id, and the place in its share
    auto owned = [&](int32_t id, uint32_t & j) {
        const uint32_t at = (uint32_t)(id + shift), gr = at / LG_GRANULE;
        j = (gr >> a.log_cluster) * LG_GRANULE + at % LG_GRANULE;
        return (gr & ((1u << a.log_cluster) - 1u)) == rank;
    };
    // The share starts on its way to the L2 cache now, so that DRAM works while the ids are counted
    // (a hint: what an earlier kernel still writes is read after the wait).
    for (int32_t g = tid; g < a.granules; g += LG_THREADS) {
        const int32_t i = token_of((uint32_t)(LG_GRANULE * g));
        if (i >= 0 && i <= n_vocab - LG_GRANULE)
            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" :: "l"(x + i), "r"(LG_GRANULE * 4) : "memory");
    }
    if (TABLE)
        for (int32_t j = tid; j < a.granules * (int)(LG_GRANULE * sizeof(T) / 16); j += LG_THREADS)
            reinterpret_cast<uint4 *>(table)[j] = make_uint4(0, 0, 0, 0);
    if (tid == 0) {
        n_list = 0;
        alb_mbar_init(&joined_bar, 1);
        alb_mbar_fence_init();
        alb_mbar_expect_tx(&joined_bar, 8u << a.log_cluster);
    }
    lg_cluster_arrive();   // CTA 0 is there to take the others' maxima
    alb_pdl_wait();
    alb_pdl_trigger();
    int32_t len = r.history_len ? r.history_len[row] : (int32_t)r.history_stride;
    bool bad = false;
    if (r.history && len > r.history_stride) { len = (int32_t)r.history_stride; bad = true; }
    if (len < 0) {   // a padding row: all CTAs of its cluster leave here
        lg_cluster_wait();
        return;
    }
    const float temp = r.temperature ? r.temperature[row] : 0.0f;
    const int64_t mask_row = !r.allow ? -1 : r.allow_row ? r.allow_row[row] : row;
    if (mask_row >= r.n_allow) bad = true;
    const bool masked = mask_row >= 0 && mask_row < r.n_allow;
    if (masked) {   // the share's bits, bit b of word 4 g + w that of place 32 w + b of granule g
        const uint32_t * allow = r.allow + mask_row * r.allow_stride;
        const int32_t last = (n_vocab - 1) >> 5;
        for (int32_t w = tid; w < a.granules * 4; w += LG_THREADS) {
            const int32_t i = token_of((uint32_t)(32 * w));   // (bits of places outside the row are not used)
            uint32_t bits = i <= n_vocab - 1 ? allow[max(i, 0) >> 5] : 0u;
            if (shift) bits = i < 0 ? bits << shift : __funnelshift_r(bits, allow[min((i >> 5) + 1, last)], i & 31);
            mask[w] = bits;
        }
    }
    __syncthreads();   // table, list and mask are set up

    RowRules k = {1.0f, 0.0f, 0.0f};
    bool listed = true;
    if (TABLE) {
        if (r.repetition) k.rep = r.repetition[row];
        if (r.frequency) k.freq = r.frequency[row];
        if (r.presence) k.pres = r.presence[row];
        if (r.bias_ids) {
            // the last entry of an id counts: blocks of entries from the back, within a block the
            // largest place wins the table entry; its thread leaves x + bias in y and a mark that
            // keeps earlier entries away
            int32_t b0 = r.bias_offsets[row], b1 = r.bias_offsets[row + 1];
            // (in order and inside the list: 0 <= b0 <= b1 <= n_bias)
            if (b0 < 0 || b1 > r.n_bias || b0 > b1) { bad = true; b0 = max(b0, 0); b1 = min(b1, r.n_bias); }
            for (int32_t end = b1; end > b0; end -= LG_THREADS) {
                const int32_t e = end - 1 - tid;
                const uint32_t place = LG_THREADS - tid;
                uint32_t j = 0;
                int32_t id = -1;
                if (e >= b0) {
                    id = r.bias_ids[e];
                    if (id >= n_vocab) { bad = true; id = -1; }
                    if (id >= 0 && (!owned(id, j) || (table[j] & Entry<T>::BIASED))) id = -1;
                }
                __syncthreads();   // marks are read before places go in
                if (id >= 0) lg_max(table, j, place);
                __syncthreads();
                const bool won = id >= 0 && table[j] == place;
                __syncthreads();
                if (won) {
                    y[id] = __fadd_rn(x[id], r.bias_values[e]);
                    table[j] = (T)Entry<T>::BIASED;
                    const uint32_t at = atomicAdd(&n_list, 1u);
                    if (at < LG_LIST) list[at] = (uint16_t)j;
                }
                __syncthreads();
            }
        }
        if (r.history) {
            const int32_t start = r.last_n > 0 && len > r.last_n ? len - r.last_n : 0;
            const int32_t prompt = r.prompt_len ? r.prompt_len[row] : 0;
            const int32_t * h = r.history + row * r.history_stride;
            auto count = [&](int32_t e, int32_t id) {
                uint32_t j;
                if (id >= n_vocab) bad = true;
                if ((uint32_t)id >= (uint32_t)n_vocab || !owned(id, j)) return;
                const uint32_t c = e < prompt ? lg_or(table, j, Entry<T>::PROMPT) : lg_add(table, j, 1u);
                if (c == 0u) {   // the first of this id
                    const uint32_t at = atomicAdd(&n_list, 1u);
                    if (at < LG_LIST) list[at] = (uint16_t)j;
                }
            };
            for (int32_t e = start + tid; e < len; e += LG_IDS * LG_THREADS) {
                int32_t id[LG_IDS];
#pragma unroll
                for (int u = 0; u < LG_IDS; ++u) id[u] = e + u * LG_THREADS < len ? h[e + u * LG_THREADS] : -1;
#pragma unroll
                for (int u = 0; u < LG_IDS; ++u)
                    if (e - tid + u * LG_THREADS < len) count(e + u * LG_THREADS, id[u]);
            }
        }
        __syncthreads();   // every id is counted
        const uint32_t n = n_list;
        listed = n <= LG_LIST;   // beyond, the counts stay in the table for the pass over the logits
        if (listed)
            for (uint32_t l = tid; l < n; l += LG_THREADS) {
                const uint32_t j = list[l], c = table[j];
                const int32_t i = token_of(j);
                settled[l + 1] = lg_penalty<T>((c & Entry<T>::BIASED) ? y[i] : x[i], c, k);
                table[j] = (T)(l + 1);
            }
        __syncthreads();   // every value is in place
    }
    const bool plain_temp = temp > 0x1p-20f && temp < 0x1p20f;
    const float inv = plain_temp ? __frcp_rn(temp) : 0.0f;
    const uint64_t inv2 = lg_pair(inv, inv), minus_temp2 = lg_pair(-temp, -temp);
    // This warp's granules are warp + 16 m of the share, lane l taking the group of four at 4 l; m from
    // m0 to m1 - 1 lie inside the row, so may one before (shift) and one behind reach over its ends.
    const int log_step = a.log_cluster + 11;
    static_assert(LG_WARPS * LG_GRANULE == 1 << 11, "tokens from a warp's granule to its next, per CTA");
    const int32_t first = token_of((uint32_t)(LG_GRANULE * warp));
    const int32_t m0 = first < 0 ? 1 : 0, m1 = n_vocab - LG_GRANULE < first ? 0 : ((n_vocab - LG_GRANULE - first) >> log_step) + 1;
    float best = -INFINITY;
    int32_t best_m = 0;    // the granule that has it
    // the rules on this lane's group of granule m
    auto rules = [&](float4 & f, int32_t m) {
        const uint32_t group = (uint32_t)(warp + LG_WARPS * m);
        if (TABLE) {
            uint32_t c[4];
            if (lg_entries(table, LG_GRANULE * group + 4 * lane, c)) {
                if (listed) {
                    const float s0 = settled[c[0]], s1 = settled[c[1]], s2 = settled[c[2]], s3 = settled[c[3]];
                    f.x = c[0] ? s0 : f.x;
                    f.y = c[1] ? s1 : f.y;
                    f.z = c[2] ? s2 : f.z;
                    f.w = c[3] ? s3 : f.w;
                } else {
                    const float * z = y + first + (m << log_step) + 4 * lane;
                    if (c[0]) f.x = lg_penalty_called<T>((c[0] & Entry<T>::BIASED) ? z[0] : f.x, c[0], k.rep, k.freq, k.pres);
                    if (c[1]) f.y = lg_penalty_called<T>((c[1] & Entry<T>::BIASED) ? z[1] : f.y, c[1], k.rep, k.freq, k.pres);
                    if (c[2]) f.z = lg_penalty_called<T>((c[2] & Entry<T>::BIASED) ? z[2] : f.z, c[2], k.rep, k.freq, k.pres);
                    if (c[3]) f.w = lg_penalty_called<T>((c[3] & Entry<T>::BIASED) ? z[3] : f.w, c[3], k.rep, k.freq, k.pres);
                }
            }
        }
        if (temp > 0.0f) {
            const float lo = fminf(fminf(fabsf(f.x), fabsf(f.y)), fminf(fabsf(f.z), fabsf(f.w)));
            const float hi = fmaxf(fmaxf(fabsf(f.x), fabsf(f.y)), fmaxf(fabsf(f.z), fabsf(f.w)));
            if (plain_temp && lo > 0x1p-100f && hi < 0x1p100f) {   // (a NaN among them stays NaN either way)
                lg_divide2(f.x, f.y, minus_temp2, inv2);
                lg_divide2(f.z, f.w, minus_temp2, inv2);
            } else {
                f.x = __fdiv_rn(f.x, temp);
                f.y = __fdiv_rn(f.y, temp);
                f.z = __fdiv_rn(f.z, temp);
                f.w = __fdiv_rn(f.w, temp);
            }
        }
        if (masked) {
            const uint32_t bits = mask[4 * group + (lane >> 3)] >> (4 * (lane & 7));
            f.x = bits & 1u ? f.x : -INFINITY;
            f.y = bits & 2u ? f.y : -INFINITY;
            f.z = bits & 4u ? f.z : -INFINITY;
            f.w = bits & 8u ? f.w : -INFINITY;
        }
        const float top = fmaxf(fmaxf(f.x, f.y), fmaxf(f.z, f.w));   // (fmaxf passes over NaN)
        best_m = top > best ? m : best_m;   // a later group wins only if it is larger: the lowest index stays
        best = fmaxf(best, top);
    };
    // a granule that reaches over the row's ends
    auto edge = [&](int32_t m) {
        const int32_t i = first + (m << log_step) + 4 * lane;
        if (i + 3 < 0 || i >= n_vocab) return;
        auto in = [&](int e) { return i + e >= 0 && i + e < n_vocab; };
        float4 f = make_float4(in(0) ? x[i] : -INFINITY, in(1) ? x[i + 1] : -INFINITY, in(2) ? x[i + 2] : -INFINITY,
                               in(3) ? x[i + 3] : -INFINITY);
        rules(f, m);
        if (in(0)) y[i] = f.x;
        if (in(1)) y[i + 1] = f.y;
        if (in(2)) y[i + 2] = f.z;
        if (in(3)) y[i + 3] = f.w;
    };
    if (first < 0) edge(0);
    {
        const float * px = x + first + 4 * lane + ((int64_t)m0 << log_step);
        float * py = y + first + 4 * lane + ((int64_t)m0 << log_step);
        const int64_t step = (int64_t)1 << log_step;
        auto put = [&](const float4 & f) {
            if (a.vec_out) {
                *reinterpret_cast<float4 *>(py) = f;
            } else {
                py[0] = f.x;
                py[1] = f.y;
                py[2] = f.z;
                py[3] = f.w;
            }
            py += step;
        };
        int32_t m = m0;
        for (; m + LG_BATCH <= m1; m += LG_BATCH) {
            float4 v[LG_BATCH];
#pragma unroll
            for (int u = 0; u < LG_BATCH; ++u) { v[u] = lg_load(px); px += step; }
#pragma unroll
            for (int u = 0; u < LG_BATCH; ++u) { rules(v[u], m + u); put(v[u]); }
        }
        for (; m < m1; ++m) {
            float4 v = lg_load(px);
            px += step;
            rules(v, m);
            put(v);
        }
    }
    if (m1 >= m0 && first + (m1 << log_step) < n_vocab) edge(m1);
    if (bad) atomicExch(a.err, ALB_DEVERR_BAD_INDEX);
    __syncwarp();
    lg_cluster_wait();
    if (a.next) {
        uint32_t best_i = 0xffffffffu;
        if (best > -INFINITY) {   // the lowest token of the group that has it (in y, where this thread wrote it)
            const int32_t i = first + (best_m << log_step) + 4 * lane;
            for (int e = 3; e >= 0; --e)
                if (i + e >= 0 && i + e < n_vocab && y[i + e] == best) best_i = (uint32_t)(i + e);
        }
        // largest value, then lowest index; 0xffffffff where nothing beats -INFINITY
        const uint32_t none = lg_order(-INFINITY);
        uint32_t key = lg_order(best), top = __reduce_max_sync(0xffffffffu, key);
        uint32_t at = __reduce_min_sync(0xffffffffu, key == top ? best_i : 0xffffffffu);
        if (lane == 0) { red_v[warp] = top; red_i[warp] = at; }
        __syncthreads();
        if (warp == 0) {
            key = lane < LG_WARPS ? red_v[lane] : none;
            top = __reduce_max_sync(0xffffffffu, key);
            at = __reduce_min_sync(0xffffffffu, key == top && lane < LG_WARPS ? red_i[lane] : 0xffffffffu);
            if (lane == 0) lg_send(lg_remote(&joined[rank], 0), lg_remote(&joined_bar, 0), top, at);
            if (rank == 0) {
                if (!alb_mbar_wait(&joined_bar, 0)) atomicExch(a.err, ALB_DEVERR_MBAR_TIMEOUT);
                const uint2 j = lane < 1 << a.log_cluster ? joined[lane] : make_uint2(none, 0xffffffffu);
                top = __reduce_max_sync(0xffffffffu, j.x);
                at = __reduce_min_sync(0xffffffffu, j.x == top ? j.y : 0xffffffffu);
                if (lane == 0) a.next[row] = (int32_t)at;
            }
        }
    }
}

template <typename T, bool TABLE, int PER_SM>
cudaError_t launch_logits(const LogitsArgs & a, int64_t rows, cudaStream_t st) {
    const size_t smem = (size_t)a.granules * LG_GRANULE * (TABLE ? sizeof(T) : 0) + (a.r.allow ? (size_t)a.granules * 16 : 0);
    const unsigned cluster = 1u << a.log_cluster;
    static std::atomic<bool> wide_clusters[64];   // per device: clusters of 16 are allowed
    cudaError_t e = ensure_smem(k_logits<T, TABLE, PER_SM>, smem + LG_STATIC);   // the limit holds for both kinds together
    int dev = 0;
    if (e == cudaSuccess && cluster > 8) e = cudaGetDevice(&dev);
    if (e == cudaSuccess && cluster > 8 && (dev >= 64 || !wide_clusters[dev].load(std::memory_order_acquire))) {
        e = cudaFuncSetAttribute(k_logits<T, TABLE, PER_SM>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e == cudaSuccess && dev < 64) wide_clusters[dev].store(true, std::memory_order_release);
    }
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
    return cudaLaunchKernelEx(&cfg, k_logits<T, TABLE, PER_SM>, a);
}

}  // namespace

extern "C" int alb_logits_process(const float * logits, int64_t rows, int64_t n_vocab, int64_t stride,
                                  const alb_logits_rules * rules, float * out, int64_t out_stride,
                                  int32_t * next_token, void * stream) {
    ALB_CHECK_ARG(logits && rules && out && rows > 0 && rows < ((int64_t)1 << 24));
    ALB_CHECK_ARG(n_vocab > 0 && n_vocab <= 450000);   // 16 CTAs hold 32-bit counts in shared memory, places in 16 bits
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
    ALB_CHECK_ARG((((uintptr_t)next_token | (uintptr_t)r.history | (uintptr_t)r.history_len | (uintptr_t)r.prompt_len |
                    (uintptr_t)r.repetition | (uintptr_t)r.frequency | (uintptr_t)r.presence | (uintptr_t)r.temperature |
                    (uintptr_t)r.bias_offsets | (uintptr_t)r.bias_ids | (uintptr_t)r.bias_values | (uintptr_t)r.allow |
                    (uintptr_t)r.allow_row) & 3) == 0);
    LogitsArgs a = {};
    a.x = logits; a.y = out; a.n_vocab = n_vocab; a.x_stride = xs; a.y_stride = ys; a.next = next_token; a.r = r;
    if (!r.repetition && !r.frequency && !r.presence) a.r.history = nullptr;   // nothing asks for the counts
    if (!a.r.history) a.r.history_stride = 0;
    if (r.allow && !r.allow_stride) a.r.allow_stride = (n_vocab + 31) / 32;
    const bool table = a.r.history || r.bias_ids;
    // every row starts on the same 16-byte phase in x and y (or all by four bytes)
    a.vec_out = (((uintptr_t)logits ^ (uintptr_t)out) & 15) == 0 && (rows == 1 || ((xs ^ ys) & 3) == 0);
    // counts below 2^14 fit 16-bit entries
    const int64_t most = r.last_n > 0 && r.last_n < a.r.history_stride ? r.last_n : a.r.history_stride;
    const bool wide = most >= (1 << 14);
    const int64_t granules = (n_vocab + 3 + LG_GRANULE - 1) / LG_GRANULE;   // + 3: the first place may lie before the row
    // CTAs per row: enough that a share is at most 20000 tokens (its table leaves room for three CTAs an SM);
    // more while the rows do not fill the SMs and a share is worth a CTA's fixed cost
    const int64_t room = wide ? 10000 : 20000;
    a.log_cluster = 0;
    while (a.log_cluster < 4 && ((n_vocab >> a.log_cluster) > room ||
                                 ((rows << a.log_cluster) < alb_sm_count() && (n_vocab >> a.log_cluster) > 4096)))
        ++a.log_cluster;
    a.granules = (int32_t)((granules + (1 << a.log_cluster) - 1) >> a.log_cluster);
    a.err = device_error_ptr();
    ALB_CUDA_TRY(a.err ? cudaSuccess : cudaErrorMemoryAllocation);
    // a call that two CTAs an SM hold runs with the registers that leaves (64 rows of 32003 with histories
    // to 8192: 13.2 us against 18.4); where CTAs queue up a third one is worth more (256 rows of 151936:
    // 83 us against 97)
    const bool roomy = (rows << a.log_cluster) <= 2 * alb_sm_count();
    auto * f = !table ? (roomy ? launch_logits<uint16_t, false, 2> : launch_logits<uint16_t, false, 3>)
               : wide ? (roomy ? launch_logits<uint32_t, true, 2> : launch_logits<uint32_t, true, 3>)
                      : (roomy ? launch_logits<uint16_t, true, 2> : launch_logits<uint16_t, true, 3>);
    ALB_CUDA_TRY(f(a, rows, (cudaStream_t)stream));
    return ALB_OK;
}
