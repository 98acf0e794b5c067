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
    // the attention moves cells' places between lanes as 32-bit numbers of this unit
    uint32_t page_units, cell_units, unit_bytes;
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
// One warp per four heads of a token, N = D/32 neighbouring values of each per
// lane, so that the NEOX partner d +- D/2 of every value is the same slot of lane
// ^ 16.  The arithmetic is k_qk_norm_rope_kv's: fp32 squares summed in double
// (certified to round to the sequential sum's mean), then the fp32 products in
// its order.  The four sums are folded together (half the lanes keep two of them,
// a quarter one): 6 exchanges instead of 20, and the eight lanes that end with a
// head's sum find its scale, all four heads at once.
// Bound by HBM on prompts: 8192 tokens of 32 / 8 heads move 373 MB in 68 us, 84 %
// of the measured copy rate (one head a warp, with a division for the token: 136
// us; blocks of four warps 73 us, of one 102 us).  A decode step is its launch
// and four dependent loads, 2.6 us.
constexpr int AP_HEADS = 4, AP_WARPS = 2;
template <int D, bool BF16>
__global__ void __launch_bounds__(32 * AP_WARPS)
k_qk_norm_rope_kv_paged(const float * __restrict__ qkv, int64_t qkv_stride, int Hq, const float * __restrict__ qn_w,
                        const float * __restrict__ kn_w, float eps, const float * __restrict__ rope, int32_t max_pos,
                        const int32_t * __restrict__ positions, const int32_t * __restrict__ seqs, PagedView kv,
                        float * __restrict__ q_out, int * err) {
    constexpr int N = D / 32;
    using F = typename Vec<N>::F;
    const int lane = threadIdx.x & 31;
    const int64_t t = blockIdx.x;
    const int head0 = (blockIdx.y * AP_WARPS + (threadIdx.x >> 5)) * AP_HEADS, H = Hq + 2 * kv.Hkv;
    alb_pdl_wait();
    alb_pdl_trigger();
    if (head0 >= H) return;   // (a whole warp; no block barrier follows)
    const int32_t pos = positions[t];
    const int32_t seq = seqs ? seqs[t] : (t < kv.n_seqs ? (int32_t)t : kv.n_seqs);
    const float * src = qkv + t * qkv_stride + (int64_t)head0 * D + N * lane;
    float x[AP_HEADS][N];
#pragma unroll
    for (int u = 0; u < AP_HEADS; ++u) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[u][i] = 0.0f;
        if (head0 + u < H) *reinterpret_cast<F *>(x[u]) = *reinterpret_cast<const F *>(src + u * D);
    }
    if (pos < 0 || seq < 0) return;
    const bool in_table = pos < max_pos && seq < kv.n_seqs && page_of(kv, pos) < kv.max_pages;
    const int64_t cell = in_table ? cell_offset(kv, kv.table + (int64_t)seq * kv.table_stride, pos) : -1;
    if (cell < 0) {
        if (lane == 0) atomicExch(err, ALB_DEVERR_BAD_INDEX);
        return;
    }
    if (head0 < Hq + kv.Hkv) {
        float cs[2 * N];
        const float * r = rope + (int64_t)pos * D + 2 * N * (lane & 15);
        *reinterpret_cast<F *>(cs) = *reinterpret_cast<const F *>(r);
        *reinterpret_cast<F *>(cs + N) = *reinterpret_cast<const F *>(r + N);
        double s[AP_HEADS];
#pragma unroll
        for (int u = 0; u < AP_HEADS; ++u) {
            s[u] = 0.0;
#pragma unroll
            for (int i = 0; i < N; ++i) s[u] += (double)__fmul_rn(x[u][i], x[u][i]);
        }
        // lanes with bit 4 keep heads 2 and 3, then lanes with bit 3 the second of their two
        const bool up = lane & 16, odd = lane & 8;
        double a = up ? s[2] : s[0], b = up ? s[3] : s[1];
        a += __shfl_xor_sync(0xffffffffu, up ? s[0] : s[2], 16);
        b += __shfl_xor_sync(0xffffffffu, up ? s[1] : s[3], 16);
        double sum = odd ? b : a;
        sum += __shfl_xor_sync(0xffffffffu, odd ? a : b, 8);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const int mine = head0 + (lane >> 3);   // the head whose sum this lane has
        float mean;
        if (!alb_rms_mean_cert(sum, D, 1.0 / D, mean) && mine < Hq + kv.Hkv)   // the reference's sequential sum
            mean = (float)(alb_rms_seq_sum(qkv + t * qkv_stride + (int64_t)mine * D, D) / (double)D);
        const float scale = 1.0f / sqrtf(__fadd_rn(mean, eps));
        __syncwarp();
#pragma unroll
        for (int u = 0; u < AP_HEADS; ++u) {
            const int head = head0 + u;
            const float sc = __shfl_sync(0xffffffffu, scale, 8 * u);
            if (head >= Hq + kv.Hkv) continue;
            const float * w = head < Hq ? qn_w : kn_w;
            if (w) {
                float wv[N];
                *reinterpret_cast<F *>(wv) = *reinterpret_cast<const F *>(w + N * lane);
#pragma unroll
                for (int i = 0; i < N; ++i) x[u][i] = __fmul_rn(__fmul_rn(x[u][i], sc), wv[i]);
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float y = __shfl_xor_sync(0xffffffffu, x[u][i], 16);
                x[u][i] = up ? __fadd_rn(__fmul_rn(y, cs[2 * i + 1]), __fmul_rn(x[u][i], cs[2 * i]))
                             : __fsub_rn(__fmul_rn(x[u][i], cs[2 * i]), __fmul_rn(y, cs[2 * i + 1]));
            }
        }
    }
#pragma unroll
    for (int u = 0; u < AP_HEADS; ++u) {
        const int head = head0 + u;
        if (head < Hq) {
            *reinterpret_cast<F *>(q_out + (t * Hq + head) * D + N * lane) = *reinterpret_cast<F *>(x[u]);
        } else if (head < H) {
            const bool is_k = head < Hq + kv.Hkv;
            const int h = head - Hq - (is_k ? 0 : kv.Hkv);
            uint16_t * dst = (is_k ? kv.k : kv.v) + cell + (int64_t)h * kv.head_stride + N * lane;
            uint32_t out[N / 2];
#pragma unroll
            for (int i = 0; i < N; i += 2)
                out[i / 2] = (uint32_t)to_cache<BF16>(x[u][i]) | ((uint32_t)to_cache<BF16>(x[u][i + 1]) << 16);
            if (N == 4) *reinterpret_cast<uint2 *>(dst) = make_uint2(out[0], out[N / 2 - 1]);
            else        *reinterpret_cast<uint32_t *>(dst) = out[0];
        }
    }
}

// ---------------------------------------------------------------- attention
// One pass over the cells with the running maximum and sum of a softmax, on the
// tensor cores (mma m16n8k16, fp32 accumulators), everything in registers.  Up to
// 8 query heads share each byte, so the bytes bound the time and a fifth of the
// rate of these warp-level products is needed; a tcgen05 tile of 128 rows would
// hold the same 8 heads and want K and V in shared memory first.
//
// A unit is (row, K/V head, group of up to 8 query heads; 16 where more share
// the K/V head).  Its cells come in
// tiles of 16 (D = 128) or 32, and all tiles of all units, each unit's led by a
// few that stand for its setup, form one line that is cut into equal ranges, one
// per CTA (k_paged_attn): uneven lengths and few rows load the SMs alike, and
// nothing depends on the lengths but device code.  In a CTA's segment of a unit
// warp w takes every fourth tile; the warps join through shared memory, and the
// pieces of a unit that a range's border cuts are joined by k_paged_attn_join.
//
// Score product, S = Q K^T:  A (16 x 16) holds the 8 heads twice, rows 0-7 the
// leading 11 bits of q and rows 8-15 the rest, so one instruction gives both
// parts of S and c[0] + c[2], c[1] + c[3] their sum: q keeps 22 bits and more at
// no extra instruction.  bf16 caches need three parts of 8 bits: up to four heads
// have them in rows 0-3, 4-7 and 8-11 (FOUR), more take a second product.  Each row of q is scaled by a power of two first, so that its
// largest value has 10 bits before the point and no part underflows.
// Value product, O = P V:  the accumulator layout of S is the A layout of P, so
// the probabilities never leave their registers; they too are split in rows 0-7
// and 8-15.  Both products sum over an index whose order is free, so the loads
// pick it: a lane's 16-byte load of K (8 neighbouring values) feeds two k steps,
// and of V eight n columns (values 8 g + j of a 64-value half, j = column tile).
// The value product starts from zero for every tile and is added to the sums
// in fp32 rounding to nearest: the tensor cores truncate when they accumulate,
// which a long chain would gather into a bias.
//
// Exponents are base 2 and the running maximum is rounded up to a whole number,
// so rescaling is exact.  fp16 probabilities are scaled by 2^15 to stay clear of
// fp16's subnormals (p >= 2^-24 of the largest keeps its leading part normal).
// bf16 has fp32's exponents: its values may be as large as the sums can be, so its
// probabilities are scaled by 2^-k where a row has at most 2^k cells (table and
// window say so), and no sum passes the largest |V|; q is scaled below 2^-9, so
// that 128 products with any K fit too.
//
// Bound by HBM: 48 sequences of 8k to 32k cells (32 / 8 heads of 128) stream 6.6 to
// 6.75 TB/s, 4.2 GB in 622 us (lengths drawn anew hold 3.8 to 4.4 GB: 575 to 664
// us and more); 37 ragged ones take 109 us (bf16, its three parts in one product for up to
// four heads).  bf16 with five to eight heads a group takes two products and keeps
// the third parts of q in shared memory: 64 sequences of 4k to 8k cells 303 us, 5.3
// TB/s (4.3 with all parts in registers), where four heads stream 6.6.  Units of 16
// heads take one product a part of all 16: 200 sequences of 4k to 8k cells with
// 16 / 1 heads 136 us in fp16, 4.6 TB/s, and 154 in bf16 (two units of eight, which
// read K and V twice: 183 and 226).
//
// A warp has a tile of K and V (8 KB) in flight while it works on the one before,
// twelve warps an SM 96 KB; 16 warps at 128 registers spill (907 us for the 48
// sequences), eight at 255 hold too little (676 us), which is what units of 16 run
// with: 64 KB an SM in flight for two thirds of the rate.  At D = 128 all kinds
// spill a little: 36 bytes a thread for bf16 with up to four heads, 44 for fp16, 80
// for bf16 of 16 heads and 128 of five to eight (at D = 64 none).  K through the L1
// cache, whose half lines the next load takes, is worth a tenth on short calls.  Few
// rows are bound by the chain of dependent loads (lengths, page, K and V; the join:
// what is unfinished, its pieces): one sequence of 640 cells 8.2 us (bf16 8.4), of
// 32768 cells 32 us, 200 windows of single cells 22 us.  A unit's setup weighs six
// tiles (0: 29 us for the windows and 122 for the ragged batch, 12: 22.8 and 110).
constexpr int PA_WARPS = 4;
constexpr int PA_THREADS = 32 * PA_WARPS;
// CTAs per SM: what the registers allow (168 a thread for units of 8 heads, 255 for units of 16)
template <int R> constexpr int PA_CTAS_PER_SM = R == 1 ? 3 : 2;
// Cells of a tile: 16 per product step, 8 KB of K and V in a warp's registers either way.
template <int D> constexpr int PA_TILE = 16 * 128 / D;
constexpr int PA_MAX_CTAS = 1024;        // of units of 8 heads; of 16: half as many
constexpr int PA_MIN_TILES = 4;          // a CTA's range is at least a tile per warp
constexpr int PA_SETUP = 6;              // what a unit costs beside its tiles, in tiles
template <bool BF16> constexpr float PA_SHIFT = BF16 ? 0.0f : 15.0f;     // of the probabilities' exponents
template <bool BF16> constexpr int PA_Q_EXP = BF16 ? -10 : 9;            // of a row of q's largest value

// What each CTA left unfinished: the unit that its range began and did not end
// (its tail; row -1: none), and whether the unit that its range began inside of
// (its head) ends there.
// The pieces' maxima and sums by head, [0] the CTA's head, [1] its tail.
struct PaMeta {
    int32_t tail_row[PA_MAX_CTAS], tail_unit[PA_MAX_CTAS], head_ends[PA_MAX_CTAS];
    float m[2][16][PA_MAX_CTAS], l[2][16][PA_MAX_CTAS];
};
// A piece's sums: [8 R heads][D], head of CTA c at place 2 c, its tail at 2 c + 1.
template <int D, int R> __host__ __device__ constexpr size_t pa_piece_floats() { return (size_t)8 * R * D; }

struct PaArgs {
    const float * q;
    PagedView kv;
    const int32_t * seqs, * lengths;
    int64_t n_rows;
    int32_t Hq, G, groups, window;
    float scale_log2;
    float p_scale;       // what probabilities and their sums are scaled by: 2^PA_SHIFT (fp16), 2^-k
    PaMeta * meta;
    float * pieces;
    float * out, * lse;
    int * err;
};

// The positions [lo, hi) row r sees; `bad`: its sequence or length was out of range.
__device__ __forceinline__ void pa_span(const PaArgs & a, int64_t r, int32_t & lo, int32_t & hi, int32_t & seq, bool & bad) {
    hi = a.lengths[r];
    seq = a.seqs ? a.seqs[r] : (r < a.kv.n_seqs ? (int32_t)r : -1);
    lo = 0;
    bad = false;
    if (hi <= 0) { hi = 0; return; }
    const int64_t most = (int64_t)a.kv.max_pages * a.kv.page_size;
    if ((uint32_t)seq >= (uint32_t)a.kv.n_seqs) { hi = 0; bad = true; }
    else if (hi > most) { hi = (int32_t)most; bad = true; }
    if (a.window > 0 && hi > a.window) lo = hi - a.window;
}
template <int TILE> __device__ __forceinline__ int32_t pa_tiles(const PaArgs & a, int64_t r) {
    int32_t lo, hi, seq;
    bool bad;
    pa_span(a, r, lo, hi, seq, bad);
    return (int32_t)(((uint32_t)(hi - lo) + TILE - 1) / TILE);
}

// What a unit of row r weighs on the line: its tiles, and the work that any unit is.
template <int TILE> __device__ __forceinline__ int32_t pa_weight(const PaArgs & a, int64_t r) {
    const int32_t n = pa_tiles<TILE>(a, r);
    return n ? n + PA_SETUP : 0;
}

// 1 / p_scale, both powers of two.
__device__ __forceinline__ float pa_unscale(const PaArgs & a) { return __uint_as_float(0x7f000000u - __float_as_uint(a.p_scale)); }

__device__ __forceinline__ float pa_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ const uint4 pa_zeros[16] = {};   // what a cell that is not seen reads instead

// 16 bytes of K: an instruction takes 64 bytes from each of 8 cells, so its line
// stays in the L1 cache for the next one.
__device__ __forceinline__ uint4 pa_load_k(const uint16_t * p) {
    uint4 r;
    asm volatile("ld.global.nc.L1::evict_first.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
    return r;
}
// 16 bytes of V: an instruction takes whole lines.
__device__ __forceinline__ uint4 pa_load_v(const uint16_t * p) {
    uint4 r;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
    return r;
}
template <bool BF16>
__device__ __forceinline__ void pa_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same from zero.
template <bool BF16>
__device__ __forceinline__ void pa_mma0(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
// x and y as packed 16-bit parts of falling weight; each part is the rounding of
// what the ones before it left (exact differences).
template <bool BF16>
__device__ __forceinline__ void pa_split(float x, float y, uint32_t & hi, uint32_t & mid, uint32_t & lo) {
    if (BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        const float2 hf = __bfloat1622float2(h);
        const float x1 = x - hf.x, y1 = y - hf.y;
        const __nv_bfloat162 m = __floats2bfloat162_rn(x1, y1);
        const float2 mf = __bfloat1622float2(m);
        const __nv_bfloat162 l = __floats2bfloat162_rn(x1 - mf.x, y1 - mf.y);
        hi = *reinterpret_cast<const uint32_t *>(&h);
        mid = *reinterpret_cast<const uint32_t *>(&m);
        lo = *reinterpret_cast<const uint32_t *>(&l);
    } else {
        const __half2 h = __floats2half2_rn(x, y);
        const float2 hf = __half22float2(h);
        const __half2 m = __floats2half2_rn(x - hf.x, y - hf.y);
        hi = *reinterpret_cast<const uint32_t *>(&h);
        mid = *reinterpret_cast<const uint32_t *>(&m);
        lo = 0;
    }
}

// R: heads of a unit / 8.  R = 1 has two parts of its 8 heads in a product's 16
// rows (FOUR: three parts of up to 4), R = 2 a part of 16 heads, product by product.
template <int D, bool BF16, bool FOUR, int R>
__global__ void __launch_bounds__(PA_THREADS, PA_CTAS_PER_SM<R>)
k_paged_attn(const __grid_constant__ PaArgs a) {
    constexpr int KL = D / 32, VH = D / 64;       // 16-byte loads of K per cell and lane; 64-value halves of V
    constexpr int TILE = PA_TILE<D>, SUB = TILE / 16;
    constexpr int PITCH = D + 4;
    // Parts of q that do not stay in registers (they would spill), a lane's own: the third for R = 1
    // with bf16 of more than four heads, all but the first for R = 2.
    constexpr int PARTS = BF16 ? 3 : 2, REST = R == 2 ? 2 * (PARTS - 1) : BF16 && !FOUR ? 1 : 0;
    constexpr size_t SO = (size_t)PA_WARPS * 8 * R * PITCH * 4, SQ = (size_t)PA_WARPS * REST * KL * 512;
    __shared__ __align__(16) uint8_t shared[(R == 1 ? SO + SQ : SO > SQ ? SO : SQ)];   // R = 2: one after the other
    float (* so)[8 * R][PITCH] = reinterpret_cast<float (*)[8 * R][PITCH]>(shared);
    uint4 (* sq)[REST ? REST : 1][KL][32] = reinterpret_cast<uint4 (*)[REST ? REST : 1][KL][32]>(shared + (R == 1 ? SO : 0));
    __shared__ float sm[PA_WARPS][8 * R], sl[PA_WARPS][8 * R];
    __shared__ int64_t warp_sum[PA_WARPS];
    __shared__ int32_t at_row, at_unit, at_tile;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int cta = blockIdx.x;
    alb_pdl_wait();
    alb_pdl_trigger();   // the join may take its place; it waits for this grid's end

    // ---- the plan: this CTA's range of the line of tiles
    const int32_t units = a.kv.Hkv * a.groups;
    const int64_t per_thread = (a.n_rows + PA_THREADS - 1) / PA_THREADS;
    const int64_t r0 = tid * per_thread, r1 = min(a.n_rows, r0 + per_thread);
    int64_t mine = 0;
    for (int64_t r = r0; r < r1; ++r) mine += pa_weight<TILE>(a, r);
    int64_t scan = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= o) scan += v;
    }
    if (lane == 31) warp_sum[warp] = scan;
    __syncthreads();
    int64_t before = scan - mine, total = 0;
#pragma unroll
    for (int w = 0; w < PA_WARPS; ++w) {
        if (w < warp) before += warp_sum[w];
        total += warp_sum[w];
    }
    before *= units;
    total *= units;
    const int64_t want = (total + PA_MIN_TILES - 1) / PA_MIN_TILES;
    const int64_t ctas = want < gridDim.x ? want : gridDim.x;
    int64_t start = 0, left = 0;
    if (cta < ctas) {
        const int64_t each = total / ctas, more = total - each * ctas;
        start = cta * each + (cta < more ? cta : more);
        left = each + (cta < more ? 1 : 0);
    }
    if (left > 0 && start >= before && start < before + mine * units) {
        int64_t rem = start - before;
        int64_t r = r0;
        for (;; ++r) {
            const int64_t here = (int64_t)pa_weight<TILE>(a, r) * units;
            if (rem < here) break;
            rem -= here;
        }
        const int32_t n = pa_weight<TILE>(a, r);
        at_row = (int32_t)r;
        at_unit = (int32_t)(rem / n);
        at_tile = (int32_t)(rem % n) - PA_SETUP;
    }
    __syncthreads();
    int32_t tail_row = -1, tail_unit = 0, head_ends = 0;
    int32_t row = at_row, unit = at_unit, tile = at_tile;

    // ---- rows that see nothing, dealt out over the CTAs; rows out of range are reported
    for (int64_t r = cta; r < a.n_rows; r += gridDim.x) {
        int32_t lo, hi, seq;
        bool bad;
        pa_span(a, r, lo, hi, seq, bad);
        if (bad && tid == 0) atomicExch(a.err, ALB_DEVERR_BAD_INDEX);
        if (hi > lo || a.lengths[r] < 0) continue;
        float * o = a.out + r * a.Hq * D;
        for (int i = tid; i < a.Hq * D / 4; i += PA_THREADS) reinterpret_cast<float4 *>(o)[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (a.lse)
            for (int i = tid; i < a.Hq; i += PA_THREADS) a.lse[r * a.Hq + i] = -INFINITY;
    }

    // ---- the segments
    while (left > 0) {
        int32_t lo, hi, seq;
        bool bad;
        pa_span(a, row, lo, hi, seq, bad);
        const int32_t all = (int32_t)(((uint32_t)(hi - lo) + TILE - 1) / TILE);
        const int32_t take = (int32_t)min((int64_t)(all - tile), left);
        left -= take;
        if (tile + take <= 0) break;         // the range ends in the unit's setup, which is the next one's then
        const bool begins = tile <= 0, ends = tile + take == all;
        const int32_t n = begins ? tile + take : take;
        lo += max(tile, 0) * TILE;
        const int32_t kvh = unit / a.groups, grp = unit - kvh * a.groups;
        const int heads = min(8 * R, a.G - 8 * R * grp);
        const int32_t head0 = kvh * a.G + 8 * R * grp;
        const int gh = FOUR ? g & 3 : g;   // this lane's head
        const int32_t * table = a.kv.table + (int64_t)seq * a.kv.table_stride;
        const uint8_t * kb = reinterpret_cast<const uint8_t *>(a.kv.k + (int64_t)kvh * a.kv.head_stride + 8 * t);
        const uint8_t * vb = reinterpret_cast<const uint8_t *>(a.kv.v + (int64_t)kvh * a.kv.head_stride + 8 * g);
        const uint8_t * zeros = reinterpret_cast<const uint8_t *>(pa_zeros);

        // lane l looks after cell l % TILE of a tile: its page one tile ahead
        auto page_at = [&](int32_t i, int32_t & pos) {
            pos = lo + i * TILE + (lane & (TILE - 1));
            if (i >= n || pos >= hi) { pos = -1; return 0; }
            return __ldg(table + page_of(a.kv, pos));
        };
        auto offset_of = [&](int32_t page, int32_t pos) -> uint32_t {
            if (pos < 0) return 0xffffffffu;
            if ((uint32_t)page >= (uint32_t)a.kv.n_pages) { atomicExch(a.err, ALB_DEVERR_BAD_INDEX); return 0xffffffffu; }
            return (uint32_t)page * a.kv.page_units + (uint32_t)(pos - page_of(a.kv, pos) * a.kv.page_size) * a.kv.cell_units;
        };
        int32_t pos, pos2;
        int32_t page = page_at(warp, pos);
        int32_t page2 = page_at(warp + PA_WARPS, pos2);

        // q of head g (and g + 8): its values 32 i + 8 t .. + 7 are k steps 2 i and 2 i + 1 of this lane
        float qv[R][KL][8];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float * qr = a.q + ((int64_t)row * a.Hq + head0 + gh + 8 * r) * D + 8 * t;
#pragma unroll
            for (int i = 0; i < KL; ++i) {
#pragma unroll
                for (int e = 0; e < 8; ++e) qv[r][i][e] = 0.0f;
                if (gh + 8 * r < heads) {
                    *reinterpret_cast<float4 *>(qv[r][i]) = *reinterpret_cast<const float4 *>(qr + 32 * i);
                    *reinterpret_cast<float4 *>(qv[r][i] + 4) = *reinterpret_cast<const float4 *>(qr + 32 * i + 4);
                }
            }
        }
        uint4 K[SUB][2][KL], V[SUB][4][VH];
        bool ok[SUB][4];
        auto load_k = [&](uint32_t off) {
#pragma unroll
            for (int b = 0; b < SUB; ++b)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint32_t f = __shfl_sync(0xffffffffu, off, 16 * b + g + 8 * u);
                    const uint8_t * p = f != 0xffffffffu ? kb + (uint64_t)f * a.kv.unit_bytes : zeros;
#pragma unroll
                    for (int i = 0; i < KL; ++i) K[b][u][i] = pa_load_k(reinterpret_cast<const uint16_t *>(p) + 32 * i);
                }
        };
        auto load_v = [&](uint32_t off) {
#pragma unroll
            for (int b = 0; b < SUB; ++b)
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const uint32_t f = __shfl_sync(0xffffffffu, off, 16 * b + 2 * t + (u & 1) + 4 * (u & 2));
                    ok[b][u] = f != 0xffffffffu;
                    const uint8_t * p = ok[b][u] ? vb + (uint64_t)f * a.kv.unit_bytes : zeros;
#pragma unroll
                    for (int h = 0; h < VH; ++h) V[b][u][h] = pa_load_v(reinterpret_cast<const uint16_t *>(p) + 64 * h);
                }
        };
        uint32_t off = offset_of(page, pos);
        load_k(off);
        load_v(off);
        // A's rows 0-7 and 8-15 of the first product: R = 1 the first and second parts of its heads (FOUR:
        // first, second, third and nothing in fours), R = 2 the first parts of heads 0-7 and 8-15
        uint32_t qa[KL][4], qb[KL][4];
        float c[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < KL; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(qv[r][i][e]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // 2^e with top 2^e in [1, 2) 2^PA_Q_EXP; nothing to scale for 0 and what is not finite
            const int ex = (int)(__float_as_uint(top) >> 23);           // biased exponent, 0 for subnormals
            int e = ex == 255 || top == 0.0f ? 0 : 127 + PA_Q_EXP<BF16> - max(ex, 1);
            e = min(e, 126);
            if (BF16) e = max(e, -126);   // (at least -118 with fp16)
            const float up = __uint_as_float((uint32_t)(e + 127) << 23);
            c[r] = e > 0 ? a.scale_log2 * __uint_as_float((uint32_t)(127 - e) << 23) : a.scale_log2 * (1.0f / up);
#pragma unroll
            for (int i = 0; i < KL; ++i) {
                uint32_t h[4], m[4], l[4];
#pragma unroll
                for (int e2 = 0; e2 < 4; ++e2)
                    pa_split<BF16>(qv[r][i][2 * e2] * up, qv[r][i][2 * e2 + 1] * up, h[e2], m[e2], l[e2]);
#pragma unroll
                for (int e2 = 0; e2 < 4; ++e2) {
                    if (R == 2) {
                        if (r == 0) qa[i][e2] = h[e2];
                        else        qb[i][e2] = h[e2];
                    } else {
                        qa[i][e2] = FOUR && g >= 4 ? m[e2] : h[e2];
                        qb[i][e2] = !FOUR ? m[e2] : g < 4 ? l[e2] : 0u;
                    }
                }
                if (R == 2) {
                    sq[warp][r][i][lane] = make_uint4(m[0], m[1], m[2], m[3]);
                    if (BF16) sq[warp][2 + r][i][lane] = make_uint4(l[0], l[1], l[2], l[3]);
                } else if (REST) {
                    sq[warp][0][i][lane] = make_uint4(l[0], l[1], l[2], l[3]);
                }
            }
        }

        float o[VH][8][2 * R], m[R], l[R];
#pragma unroll
        for (int r = 0; r < R; ++r) { m[r] = -INFINITY; l[r] = 0.0f; }
#pragma unroll
        for (int h = 0; h < VH; ++h)
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int p = 0; p < 2 * R; ++p) o[h][j][p] = 0.0f;

        for (int32_t i = warp; i < n; i += PA_WARPS) {
            float x[R][SUB][4];   // scores of cells 16 b + 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
            for (int b = 0; b < SUB; ++b) {
                // Each product truncates its sums, so the small parts are summed apart from the first (in rows
                // 8-15 for R = 1, in sums of their own for R = 2), and chains are short: of 6000 random batches the
                // worst has outputs 6e-7 off (norm of the errors by norm of the outputs), with one chain a row 1.8e-6.
                float s[2][2][4], small[2][4];   // (two chains each, halves of the k steps)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
#pragma unroll
                    for (int k = 0; k < KL; ++k) {
                        const uint4 & w = K[b][u][k];
                        float (& sum)[4] = s[k & 1][u];
                        if (k < 2) pa_mma0<BF16>(sum, qa[k][0], qb[k][0], qa[k][1], qb[k][1], w.x, w.y);
                        else       pa_mma<BF16>(sum, qa[k][0], qb[k][0], qa[k][1], qb[k][1], w.x, w.y);
                        pa_mma<BF16>(sum, qa[k][2], qb[k][2], qa[k][3], qb[k][3], w.z, w.w);
                        if (R == 2) {
#pragma unroll
                            for (int p = 0; p < PARTS - 1; ++p) {
                                const uint4 y = sq[warp][2 * p][k][lane], z = sq[warp][2 * p + 1][k][lane];
                                if (k == 0 && p == 0) pa_mma0<BF16>(small[u], y.x, z.x, y.y, z.y, w.x, w.y);
                                else                  pa_mma<BF16>(small[u], y.x, z.x, y.y, z.y, w.x, w.y);
                                pa_mma<BF16>(small[u], y.z, z.z, y.w, z.w, w.z, w.w);
                            }
                        } else if (REST) {
                            const uint4 y = sq[warp][0][k][lane];
                            pa_mma<BF16>(sum, 0u, y.x, 0u, y.y, w.x, w.y);
                            pa_mma<BF16>(sum, 0u, y.z, 0u, y.w, w.z, w.w);
                        }
                    }
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const float (& s0)[4] = s[0][u >> 1], (& s1)[4] = s[1][u >> 1];
                    const int p = u & 1;
                    if (R == 2) {
                        x[0][b][u] = (s0[p] + s1[p]) + small[u >> 1][p];
                        x[R - 1][b][u] = (s0[2 + p] + s1[2 + p]) + small[u >> 1][2 + p];
                    } else {
                        x[0][b][u] = (s0[p] + s1[p]) + (s0[2 + p] + s1[2 + p]);
                    }
                }
            }
            // the next tile's K comes while this tile's softmax and values are worked on
            off = offset_of(page2, pos2);
            load_k(off);
            page2 = page_at(i + 2 * PA_WARPS, pos2);

            float fix[R];
            uint32_t part[PARTS][R][SUB][2];   // of the probabilities, by weight
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float top = -INFINITY;
#pragma unroll
                for (int b = 0; b < SUB; ++b)
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        if (FOUR) x[r][b][u] += __shfl_xor_sync(0xffffffffu, x[r][b][u], 16);   // the parts in rows g and g + 4
                        top = fmaxf(top, ok[b][u] ? __fmul_rn(x[r][b][u], c[r]) : -INFINITY);
                    }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float mn = fmaxf(m[r], ceilf(top));
                const float base = mn == -INFINITY ? 0.0f : mn;
                fix[r] = pa_ex2(m[r] - base);
                m[r] = mn;
                // one rounding from the score on, as long as the maximum of the rounded products is
                // within 2^-8 of the exact ones' (2^16 has steps of 2^-7); the rounded products beyond
                const bool big = !(fabsf(base) < 65536.0f);
                l[r] *= fix[r];
#pragma unroll
                for (int b = 0; b < SUB; ++b) {
                    float (& y)[4] = x[r][b];
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        y[u] = !ok[b][u] ? 0.0f : pa_ex2(big ? __fmul_rn(y[u], c[r]) - base + PA_SHIFT<BF16> : fmaf(y[u], c[r], PA_SHIFT<BF16> - base));
                    if (BF16)
#pragma unroll
                        for (int u = 0; u < 4; ++u) y[u] *= a.p_scale;
                    l[r] += (y[0] + y[1]) + (y[2] + y[3]);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        uint32_t last;
                        pa_split<BF16>(y[2 * u], y[2 * u + 1], part[0][r][b][u], part[1][r][b][u], last);
                        if (BF16) part[PARTS - 1][r][b][u] = last;
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < VH; ++h) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t sel = (j & 1) ? 0x7632u : 0x5410u;
                    float r[4], small[4];
#pragma unroll
                    for (int b = 0; b < SUB; ++b) {
                        auto word = [&](int u) { return reinterpret_cast<const uint32_t *>(&V[b][u][h])[j >> 1]; };
                        const uint32_t b0 = __byte_perm(word(0), word(1), sel), b1 = __byte_perm(word(2), word(3), sel);
                        if (R == 2) {
#pragma unroll
                            for (int p = 0; p < PARTS; ++p) {
                                uint32_t (& y)[SUB][2] = part[p][0], (& z)[SUB][2] = part[p][R - 1];
                                float (& sum)[4] = p == 0 ? r : small;
                                if (b == 0 && p < 2) pa_mma0<BF16>(sum, y[b][0], z[b][0], y[b][1], z[b][1], b0, b1);
                                else                 pa_mma<BF16>(sum, y[b][0], z[b][0], y[b][1], z[b][1], b0, b1);
                            }
                        } else {
                            const uint32_t y0 = FOUR && g >= 4 ? part[1][0][b][0] : part[0][0][b][0];
                            const uint32_t y1 = FOUR && g >= 4 ? part[1][0][b][1] : part[0][0][b][1];
                            const uint32_t z0 = !FOUR ? part[1][0][b][0] : g < 4 ? part[PARTS - 1][0][b][0] : 0u;
                            const uint32_t z1 = !FOUR ? part[1][0][b][1] : g < 4 ? part[PARTS - 1][0][b][1] : 0u;
                            if (b == 0) pa_mma0<BF16>(r, y0, z0, y1, z1, b0, b1);
                            else        pa_mma<BF16>(r, y0, z0, y1, z1, b0, b1);
                            if (REST) pa_mma<BF16>(r, 0u, part[PARTS - 1][0][b][0], 0u, part[PARTS - 1][0][b][1], b0, b1);
                        }
                    }
                    if (R == 2) {
#pragma unroll
                        for (int p = 0; p < 4; ++p) o[h][j][p & (2 * R - 1)] = fmaf(o[h][j][p & (2 * R - 1)], fix[(p >> 1) & (R - 1)], r[p] + small[p]);
                    } else {
                        o[h][j][0] = fmaf(o[h][j][0], fix[0], r[0] + r[2]);
                        o[h][j][1] = fmaf(o[h][j][1], fix[0], r[1] + r[3]);
                    }
                }
            }
            load_v(off);
        }

        if (FOUR) {   // the middle parts' products lie with lanes of rows 4-7
#pragma unroll
            for (int h = 0; h < VH; ++h)
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int p = 0; p < 2; ++p) o[h][j][p] += __shfl_xor_sync(0xffffffffu, o[h][j][p], 16);
        }

        // ---- join the warps: thread (head, part) adds its values
        if (R == 2) __syncthreads();   // the shared parts of q make room for the sums
#pragma unroll
        for (int r = 0; r < R; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            if (t == 0) { sm[warp][g + 8 * r] = m[r]; sl[warp][g + 8 * r] = l[r]; }
#pragma unroll
            for (int h = 0; h < VH; ++h)
#pragma unroll
                for (int p = 0; p < 2; ++p)
#pragma unroll
                    for (int j = 0; j < 8; j += 4)
                        *reinterpret_cast<float4 *>(&so[warp][g + 8 * r][64 * h + 16 * t + 8 * p + j]) =
                            make_float4(o[h][j][2 * r + p], o[h][j + 1][2 * r + p], o[h][j + 2][2 * r + p], o[h][j + 3][2 * r + p]);
        }
        __syncthreads();
        {
            constexpr int N = D * R / 16, PER = 16 / R;   // values of a thread, threads of a head
            const int h = tid / PER, d = tid % PER * N;
            float M = sm[0][h];
#pragma unroll
            for (int w = 1; w < PA_WARPS; ++w) M = fmaxf(M, sm[w][h]);
            const float base = M == -INFINITY ? 0.0f : M;
            float Ls = 0.0f, acc[N];
#pragma unroll
            for (int e = 0; e < N; ++e) acc[e] = 0.0f;
#pragma unroll
            for (int w = 0; w < PA_WARPS; ++w) {
                const float f = pa_ex2(sm[w][h] - base);
                Ls = fmaf(sl[w][h], f, Ls);
#pragma unroll
                for (int e = 0; e < N; e += 4) {
                    const float4 v = *reinterpret_cast<const float4 *>(&so[w][h][d + e]);
                    acc[e] = fmaf(v.x, f, acc[e]);
                    acc[e + 1] = fmaf(v.y, f, acc[e + 1]);
                    acc[e + 2] = fmaf(v.z, f, acc[e + 2]);
                    acc[e + 3] = fmaf(v.w, f, acc[e + 3]);
                }
            }
            if (h < heads) {
                if (begins && ends) {
                    float * dst = a.out + ((int64_t)row * a.Hq + head0 + h) * D + d;
#pragma unroll
                    for (int e = 0; e < N; ++e) acc[e] = Ls != 0.0f ? acc[e] / Ls : 0.0f;
#pragma unroll
                    for (int e = 0; e < N; e += 4)
                        *reinterpret_cast<float4 *>(dst + e) = make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
                    if (a.lse && d == 0)
                        a.lse[(int64_t)row * a.Hq + head0 + h] =
                            Ls != 0.0f ? fmaf(M, 0.693147181f, logf(Ls * (BF16 ? pa_unscale(a) : 0x1p-15f))) : -INFINITY;
                } else {
                    float * piece = a.pieces + (2 * cta + (begins ? 1 : 0)) * pa_piece_floats<D, R>() + h * D + d;
#pragma unroll
                    for (int e = 0; e < N; e += 4)
                        *reinterpret_cast<float4 *>(piece + e) = make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
                    if (d == 0) { a.meta->m[begins][h][cta] = M; a.meta->l[begins][h][cta] = Ls; }
                }
            }
            if (!begins) head_ends = ends;
            else if (!ends) { tail_row = row; tail_unit = unit; }
        }
        __syncthreads();   // the shared sums are free again
        tile = -PA_SETUP;
        if (left > 0 && ++unit == units) {
            unit = 0;
            do ++row; while (pa_tiles<TILE>(a, row) == 0);
        }
    }
    if (tid == 0) {
        a.meta->tail_row[cta] = tail_row;
        a.meta->tail_unit[cta] = tail_unit;
        a.meta->head_ends[cta] = head_ends;
    }
}

// Joins the pieces of the unit that CTA blockIdx.x of k_paged_attn began and did
// not end: its tail, then the heads of the CTAs behind it up to the one that ends
// the unit.  A block takes two of the unit's heads, a head four warps, a warp
// every fourth piece and a lane D/32 neighbouring values.  What tells whether
// there is work, where it ends and what the pieces weigh is loaded at once, 32
// pieces a warp and round; the pieces' maxima are whole numbers, so rescaling is exact
// whatever the order.
constexpr int PJ_HEADS = 2, PJ_PARTS = 4, PJ_THREADS = 32 * PJ_HEADS * PJ_PARTS;
template <int D, int R>
__global__ void __launch_bounds__(PJ_THREADS)
k_paged_attn_join(const __grid_constant__ PaArgs a) {
    constexpr int N = D / 32;
    using F = typename Vec<N>::F;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hl = warp / PJ_PARTS, part = warp % PJ_PARTS, cta = blockIdx.x;
    const int h = PJ_HEADS * blockIdx.y + hl, grid = gridDim.x;
    __shared__ __align__(16) float so[PJ_HEADS][PJ_PARTS][D];
    __shared__ float sm[PJ_HEADS][PJ_PARTS], sl[PJ_HEADS][PJ_PARTS];
    alb_pdl_wait();
    // piece i's sums: the tail of this CTA, then the head of the i-th CTA behind it
    auto piece = [&](int i) { return a.pieces + (2 * (cta + i) + (i == 0 ? 1 : 0)) * pa_piece_floats<D, R>(); };
    // lane l looks after pieces PARTS l .. of a round for where the unit ends, after PARTS l + part for its weight
    int last;                 // place of the first end among this lane's, or PARTS
    float m, l;
    auto look = [&](int i0) {
        int ends[PJ_PARTS];
#pragma unroll
        for (int u = 0; u < PJ_PARTS; ++u) {
            const int c = cta + i0 + PJ_PARTS * lane + u;
            ends[u] = a.meta->head_ends[min(c, grid - 1)] | (c >= grid - 1);
            if (i0 + lane + u == 0) ends[u] = 0;   // the tail itself (CTA `cta`; a last CTA has none)
        }
        last = PJ_PARTS;
#pragma unroll
        for (int u = PJ_PARTS - 1; u >= 0; --u)
            if (ends[u]) last = u;
        const int i = i0 + PJ_PARTS * lane + part;
        m = -INFINITY;
        l = 0.0f;
        if (cta + i < grid) { m = a.meta->m[i == 0][h][cta + i]; l = a.meta->l[i == 0][h][cta + i]; }
    };
    const int32_t row = a.meta->tail_row[cta], unit = a.meta->tail_unit[cta];
    look(0);
    const int32_t kvh = unit / a.groups, grp = unit - kvh * a.groups;
    const int heads = min(8 * R, a.G - 8 * R * grp);
    if (row >= 0 && PJ_HEADS * (int)blockIdx.y < heads) {   // uniform over the block
        float M = -INFINITY, L = 0.0f, acc[N];
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] = 0.0f;
        if (h < heads) {
            for (int i0 = 0;;) {
                const uint32_t e = __ballot_sync(0xffffffffu, last < PJ_PARTS);
                const int who = e ? __ffs(e) - 1 : 31;
                const int n = e ? PJ_PARTS * who + __shfl_sync(0xffffffffu, last, who) + 1 : 32 * PJ_PARTS;   // pieces of this round
                if (PJ_PARTS * lane + part >= n) { m = -INFINITY; l = 0.0f; }
                const float Mn = fmaxf(M, alb_warp_max(m)), base = Mn == -INFINITY ? 0.0f : Mn;
                const float fix = pa_ex2(M - base), f = pa_ex2(m - base);
                L = fmaf(L, fix, alb_warp_sum(l * f));
#pragma unroll
                for (int k = 0; k < N; ++k) acc[k] *= fix;
                M = Mn;
#pragma unroll 4
                for (int k = 0; PJ_PARTS * k + part < n; ++k) {
                    const float w = __shfl_sync(0xffffffffu, f, k);
                    float v[N];
                    *reinterpret_cast<F *>(v) = *reinterpret_cast<const F *>(piece(i0 + PJ_PARTS * k + part) + h * D + N * lane);
#pragma unroll
                    for (int j = 0; j < N; ++j) acc[j] = fmaf(v[j], w, acc[j]);
                }
                if (e) break;
                i0 += 32 * PJ_PARTS;
                look(i0);
            }
        }
        *reinterpret_cast<F *>(&so[hl][part][N * lane]) = *reinterpret_cast<F *>(acc);
        if (lane == 0) { sm[hl][part] = M; sl[hl][part] = L; }
        __syncthreads();
        if (part == 0 && h < heads) {
            float top = sm[hl][0];
#pragma unroll
            for (int p = 1; p < PJ_PARTS; ++p) top = fmaxf(top, sm[hl][p]);
            const float base = top == -INFINITY ? 0.0f : top;
            L = 0.0f;
#pragma unroll
            for (int e = 0; e < N; ++e) acc[e] = 0.0f;
#pragma unroll
            for (int p = 0; p < PJ_PARTS; ++p) {
                const float f = pa_ex2(sm[hl][p] - base);
                float v[N];
                *reinterpret_cast<F *>(v) = *reinterpret_cast<const F *>(&so[hl][p][N * lane]);
                L = fmaf(sl[hl][p], f, L);
#pragma unroll
                for (int e = 0; e < N; ++e) acc[e] = fmaf(v[e], f, acc[e]);
            }
            const int64_t head = (int64_t)row * a.Hq + kvh * a.G + 8 * R * grp + h;
#pragma unroll
            for (int e = 0; e < N; ++e) acc[e] = L != 0.0f ? acc[e] / L : 0.0f;
            *reinterpret_cast<F *>(a.out + head * D + N * lane) = *reinterpret_cast<F *>(acc);
            if (a.lse && lane == 0) a.lse[head] = L != 0.0f ? fmaf(top, 0.693147181f, logf(L * pa_unscale(a))) : -INFINITY;
        }
    }
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
    else if (c->n_pages >= ((int64_t)1 << 31) || c->n_pages * c->page_size >= ((int64_t)1 << 31) || c->n_head_kv > 65535)
        why = "invalid argument: paged cache of 2^31 cells or more, or more than 65535 heads";
    else if ((int64_t)c->max_pages * c->page_size > (1 << 30))   // (positions of a tile that starts below stay below 2^31)
        why = "invalid argument: page table of more than 2^30 positions";
    else if ((uintptr_t)c->page_table & 3) why = "invalid argument: page table not 4-byte aligned";
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
    int64_t unit = 8;
    while (kv.page_stride % (2 * unit) == 0 && kv.cell_stride % (2 * unit) == 0 && unit < ((int64_t)1 << 30)) unit *= 2;
    if ((kv.n_pages - 1) * (kv.page_stride / unit) + (kv.page_size - 1) * (kv.cell_stride / unit) >= ((int64_t)1 << 32) - 1) {
        alb_set_last_error_msg("invalid argument: paged cache strides reach beyond 2^32 units of their common power of two");
        return false;
    }
    kv.page_units = (uint32_t)(kv.page_stride / unit);   // (below 2^32 unless there is one page only, which never steps)
    kv.cell_units = (uint32_t)(kv.cell_stride / unit);
    kv.unit_bytes = (uint32_t)(2 * unit);
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
    const unsigned per_token = (unsigned)(Hq + 2 * kv.Hkv + AP_HEADS * AP_WARPS - 1) / (AP_HEADS * AP_WARPS);
    return alb_launch(k_qk_norm_rope_kv_paged<D, BF16>, dim3((unsigned)T, per_token), dim3(32 * AP_WARPS), 0, st, true,
                      qkv, qkv_stride, Hq, qn, kn, eps, rope, max_pos, positions, seqs, kv, q_out, err);
}

size_t attn_ws_bytes(int D) { return sizeof(PaMeta) + 2 * PA_MAX_CTAS * 8 * (size_t)D * sizeof(float); }

template <int D, bool BF16, bool FOUR, int R>
cudaError_t launch_attn_r(PaArgs a, cudaStream_t st) {
    a.groups = (a.G + 8 * R - 1) / (8 * R);
    const int ctas = min(PA_MAX_CTAS / R, PA_CTAS_PER_SM<R> * alb_sm_count());
    cudaError_t e = alb_launch(k_paged_attn<D, BF16, FOUR, R>, dim3((unsigned)ctas), dim3(PA_THREADS), 0, st, true, a);
    if (e != cudaSuccess) return e;
    const unsigned parts = (unsigned)(min(a.G, 8 * R) + PJ_HEADS - 1) / PJ_HEADS;
    return alb_launch(k_paged_attn_join<D, R>, dim3((unsigned)ctas, parts), dim3(PJ_THREADS), 0, st, true, a);
}

template <int D, bool BF16>
cudaError_t launch_attn(PaArgs a, cudaStream_t st) {
    int64_t most = (int64_t)a.kv.max_pages * a.kv.page_size;
    if (a.window > 0 && a.window < most) most = a.window;
    int k = 0;
    while (BF16 && ((int64_t)1 << k) < most) ++k;
    a.p_scale = std::ldexp(1.0f, (int)PA_SHIFT<BF16> - k);
    // more than 8 heads a group: units of 16, which read K and V once
    if (a.G > 8) return launch_attn_r<D, BF16, false, 2>(a, st);
    return BF16 && a.G <= 4 ? launch_attn_r<D, BF16, BF16, 1>(a, st) : launch_attn_r<D, BF16, false, 1>(a, st);
}

}  // namespace

extern "C" int alb_qk_norm_rope_kv_paged(const float * qkv, int64_t qkv_stride, int64_t T, int32_t n_head,
                                         const float * q_norm, const float * k_norm, float eps,
                                         const float * rope_table, int32_t max_pos, const int32_t * positions,
                                         const int32_t * seqs, const alb_paged_kv * kv, float * q_out, void * stream) {
    PagedView v;
    if (!paged_view(kv, v, true)) return ALB_ERR_INVALID;
    ALB_CHECK_ARG(qkv && rope_table && positions && q_out && T > 0 && max_pos > 0 && eps >= 0.0f);
    ALB_CHECK_ARG(n_head > 0 && n_head <= 65535 && T < ((int64_t)1 << 31) / (n_head + 2 * v.Hkv));
    const int64_t dense = (int64_t)(n_head + 2 * v.Hkv) * kv->head_dim;
    ALB_CHECK_ARG(qkv_stride == 0 || (qkv_stride >= dense && qkv_stride % 4 == 0 && qkv_stride < ((int64_t)1 << 31)));
    ALB_CHECK_ARG((((uintptr_t)qkv | (uintptr_t)q_norm | (uintptr_t)k_norm | (uintptr_t)rope_table | (uintptr_t)q_out) & 15) == 0);
    ALB_CHECK_ARG((((uintptr_t)positions | (uintptr_t)seqs) & 3) == 0);
    // a token's queries in the place of another's heads would change them before they are read
    const int64_t stride = qkv_stride ? qkv_stride : dense;
    const uintptr_t x0 = (uintptr_t)qkv, x1 = x0 + 4 * (uintptr_t)((T - 1) * stride + dense);
    const uintptr_t y0 = (uintptr_t)q_out, y1 = y0 + 4 * (uintptr_t)(T * n_head * kv->head_dim);
    ALB_CHECK_ARG((T == 1 && qkv == q_out) || x1 <= y0 || y1 <= x0);
    int * err = device_error_ptr();
    ALB_CUDA_TRY(err ? cudaSuccess : cudaErrorMemoryAllocation);
    auto * f = kv->head_dim == 128 ? (kv->type == ALB_KV_BF16 ? launch_append<128, true> : launch_append<128, false>)
                                   : (kv->type == ALB_KV_BF16 ? launch_append<64, true> : launch_append<64, false>);
    ALB_CUDA_TRY(f(qkv, stride, T, n_head, q_norm, k_norm, eps, rope_table, max_pos,
                   positions, seqs, v, q_out, err, (cudaStream_t)stream));
    return ALB_OK;
}

extern "C" size_t alb_paged_attn_workspace_bytes(const alb_paged_kv * kv, int64_t n_rows, int32_t n_head) {
    PagedView v;
    if (!paged_view(kv, v, false) || n_rows <= 0 || n_head <= 0 || n_head % v.Hkv != 0) return 0;
    return attn_ws_bytes(kv->head_dim);
}

extern "C" int alb_paged_attn(const float * q, int64_t n_rows, int32_t n_head, const alb_paged_kv * kv,
                              const int32_t * seqs, const int32_t * lengths, int32_t window, float scale,
                              void * workspace, float * out, float * lse, void * stream) {
    PagedView v;
    if (!paged_view(kv, v, true)) return ALB_ERR_INVALID;
    ALB_CHECK_ARG(q && lengths && workspace && out && n_rows > 0 && n_rows < ((int64_t)1 << 24) && window >= 0);
    ALB_CHECK_ARG(n_head > 0 && n_head < 4096 && n_head % v.Hkv == 0);   // 2^24 rows x 2^27 tiles x 2^12 units < 2^63
    ALB_CHECK_ARG(scale > 0.0f && std::isfinite(scale));
    ALB_CHECK_ARG((((uintptr_t)q | (uintptr_t)out | (uintptr_t)workspace) & 15) == 0);
    ALB_CHECK_ARG((((uintptr_t)lengths | (uintptr_t)seqs | (uintptr_t)lse) & 3) == 0);
    // in place is fine: a unit reads its queries before it writes, and nothing else reads them
    const uintptr_t x0 = (uintptr_t)q, y0 = (uintptr_t)out, bytes = 4 * (uintptr_t)(n_rows * n_head * kv->head_dim);
    ALB_CHECK_ARG(x0 == y0 || x0 + bytes <= y0 || y0 + bytes <= x0);
    PaArgs a = {};
    a.q = q; a.kv = v; a.seqs = seqs; a.lengths = lengths; a.n_rows = n_rows; a.Hq = n_head; a.G = n_head / v.Hkv;
    a.window = window; a.scale_log2 = scale * 1.44269504f; a.out = out; a.lse = lse;
    a.meta = static_cast<PaMeta *>(workspace);
    a.pieces = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + sizeof(PaMeta));
    a.err = device_error_ptr();
    ALB_CUDA_TRY(a.err ? cudaSuccess : cudaErrorMemoryAllocation);
    auto * f = kv->head_dim == 128 ? (kv->type == ALB_KV_BF16 ? launch_attn<128, true> : launch_attn<128, false>)
                                   : (kv->type == ALB_KV_BF16 ? launch_attn<64, true> : launch_attn<64, false>);
    ALB_CUDA_TRY(f(a, (cudaStream_t)stream));
    return ALB_OK;
}
