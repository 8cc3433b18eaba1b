// The mixture-of-experts layer as one cooperative kernel, a CTA per SM.
//
// For a few tokens the layer is bound by reading the touched experts' weights once (3 x model x expert bytes each when
// gated), so everything is arranged around keeping those reads in flight:
//  0. Router: logits (an expert and 8 tokens at a time, shared by warps of a CTA), and x rewritten as digits (below).
//     Grid barrier. Every CTA then finds all tokens' experts itself, a warp per token: cheaper than another barrier; of more
//     tokens than warps, each block of 8 has been ranked by the CTA that completed its logits, before the barrier. Every CTA
//     sorts the (token, choice) pairs by expert into groups of one expert and up to 8 NT pairs.
//  1. Input products: units of one group and 16 rows of w_in (8 of each half when gated, so that a lane holds both
//     factors of a hidden value), K in chunks of 128 bytes. Grid barrier, the hidden values rewritten as digits, grid
//     barrier.
//  2. Output products: units of one group and 16 rows of w_out; weighted results per pair. Grid barrier.
//  3. The sum over each token's pairs, in the order of their rank: the result does not depend on the schedule.
// A CTA owns a contiguous range of units of equal cost (unit_cost) and its warps equal contiguous ranges of the units' chunks; a unit cut between
// warps meets through partial sums (`segments`), added by the warp that holds its start. Each warp feeds itself: a ring of
// SLOTS 2 KB boxes loaded by TMA (128-byte swizzle, no multicast), the next box issued as soon as one is in registers. The
// ring runs on into phase 2's weights, which do not depend on the barriers: DRAM stays busy while the hidden values
// are exchanged.
//
// Arithmetic: the int8 weights multiply as they are (mma.sync m16n8k32 s8, weights as the 16-row operand, 8 pairs as its
// columns). The other operand is a row of x or of hidden values in fixed point, q = rint(v 2^s) with the row's own s, cut
// into D balanced base-256 digits that are int8 operands too: every digit's sum is an exact int32 (65536 x 128 x 128 stays
// below 2^31). The lowest digit's sum over a chunk is rounded to the next digit's unit and added there, so that it needs no
// accumulators of its own: an error of a fraction of what rounding the values themselves costs, and the same one in
// whatever order the chunks come. The other digits' sums together are an exact int64. Held are 31 bits below the row's
// largest value for float16 layers (D = 4) and 39 bits for float32 ones (D = 5): the step has to be small next to the quiet
// channels of a row, not to its largest value, since an output's weights may leave the loud ones out. With a digit less (23
// and 31 bits) such outputs were off by up to 15 roundings of float16 for channels 3000 to 60000 times the others; 64 tokens
// through 6 of 64 experts (2048 x 1408) took 152 us then and 156 with one more, one token (2048 x 1024) 35.5 and 36.5.
// Measured against converting the weights to bfloat16 in registers and multiplying two or three bfloat16 pieces, with three
// digits: 239 instructions per 2 KB of weights became about 100, 8 tokens through 2 of 8 experts (4096 x 8192) went from
// 163 to 149 us (6.1 TB/s while the weights stream), 64 tokens through 6 of 64 experts from 199 to 164 us. The tensor
// cores' rate does not matter here (one token per expert uses an eighth of a tile), and 128-row tcgen05 tiles would cut the
// work too coarsely for one token.
// A token with an infinite or NaN value, or such a hidden value, gets NaN.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "og_act.cuh"
#include "og_gemm.h"
#include "og_moe.h"
#include "og_ptx.cuh"

namespace og {

namespace moe {
constexpr int CHUNK = 128;                    // bytes of K of a box
constexpr int SLOTS = 4;                      // boxes in flight per warp
constexpr int MAX_PAIRS = MOE_MAX_TOKENS * MOE_MAX_TOP_K;

// MT matrix tiles of 16 weight rows in a unit, NT tiles of 8 columns in a group. MT = 1: 16 warps (of at most 128
// registers), the finest units, for one or two tokens, whose columns are all the same few rows. MT = 2: 8 warps, each
// column digit read from L1 for 32 weight rows instead of 16: with 8 different rows a load touches 8 lines, and from
// some 4 columns on these loads, not DRAM, set the time.
//
// ALIGNED: weight rows on 16-byte boundaries, loaded by TMA. Others arrive by 16-byte asynchronous copies of the aligned
// units that hold a row's 128 bytes (nine of them), and the operands are put together from neighbouring words.
template <int NT_, int MT_, bool ALIGNED_>
struct Shape {
    static constexpr int NT = NT_, MT = MT_;
    static constexpr bool ALIGNED = ALIGNED_;
    static constexpr int PITCH = ALIGNED ? CHUNK : CHUNK + 16;  // bytes of a row in shared memory
    static constexpr int WARPS = MT == 1 ? 16 : 8;
    static constexpr int THREADS = 32 * WARPS;
    static constexpr int ROWS = 16 * MT;
    static constexpr int BOX = ROWS * PITCH;              // 2 or 4 KB (and an eighth); 128 KB of boxes in flight per SM
    static constexpr int SUMS = ROWS * 8 * NT;            // of a unit
    static constexpr int WHOLE_FROM = WARPS * 3 / 4;      // warps with a whole unit each: 96 KB in flight are enough
    static constexpr int RING = WARPS * SLOTS * BOX;
};
}  // namespace moe

struct MoeFusedParams {
    MoeLaunch L;
    int chunks_in, chunks_out;  // K chunks of the two products
    int blocks_in, blocks_out;  // units per group
    int router_split;           // warps that share one (expert, 8 tokens) of the router
    int vec;                    // rows of x and of the router allow loads of four elements
    int hidden_pitch, out_pitch;  // elements between the rows of L.hidden and L.outputs, multiples of 4
    const int8_t* end_in;       // past the last weight
    const int8_t* end_out;
};

// A group: one expert and a run of the pairs sorted by expert.
struct MoeGroup {
    uint16_t expert, first, count;
    uint16_t before;  // the cost of a unit of every group before it
};

// What a unit of a group costs next to others: its columns' digits come from L1 or L2 and cost more the more of them
// differ, and each further tile has its own loads and products. Shares of equal bytes took, in us a phase and with three
// digits: 64 tokens through 6 of 64 experts (2048 x 1408) 66 with up to 6 pairs, 71 with 7 or 8, 89 with 9 to 12 (a second
// tile); 8 tokens through 2 of 8 experts (4096 x 8192) 80 (phase 1) and 39 (2) with one pair, 88 and 48 with 2 to 4; NT = 4,
// two, three and four tiles 50, 68 and 86. With four digits the second tile of NT = 2 weighs more: the 64 tokens took 178,
// 168, 162 and 156 us with 5, 8, 11 and 14 for it, float32 ones 177, 173, 172 and 174. Read off float16 and float32 layers
// with aligned weights; the unaligned load path shares by the same numbers.
template <int NT>
__device__ __forceinline__ int unit_cost(int pairs) {
    return (pairs == 1 ? 16 : pairs <= 6 ? 18 : 20) + (pairs - 1) / 8 * (NT == 4 ? 12 : 14);
}

template <class S>
struct MoeShared {
    static constexpr int GROUPS = MOE_MAX_EXPERTS + moe::MAX_PAIRS / (8 * S::NT);
    uint64_t full[S::WARPS][moe::SLOTS];
    double logit_part[2][S::WARPS][8];
    int count[MOE_MAX_EXPERTS];        // pairs of each expert, then the place of its first one in `order`
    float weight[moe::MAX_PAIRS];      // by pair (token * top_k + rank)
    uint32_t most[moe::MAX_PAIRS];     // by pair: the bits of its largest hidden value seen by this CTA
    int16_t shift[moe::MAX_PAIRS];     // by pair: the shift of its token's x, later of its hidden values
    alignas(16) uint16_t id[moe::MAX_PAIRS];  // by pair
    uint16_t order[moe::MAX_PAIRS];    // pairs sorted by expert
    MoeGroup group[GROUPS];
    int warp_total[2][S::WARPS];
    unsigned complete;                 // token blocks whose logits this CTA completed
    int groups;
    int cost;                          // of a unit of every group
    int abort;
    int failed;
};

template <class S>
constexpr size_t moe_smem_bytes() {
    static_assert(1024 + size_t(S::RING) + sizeof(MoeShared<S>) <= 232448, "shared memory of a CTA");
    return 1024 + size_t(S::RING) + sizeof(MoeShared<S>);
}

// ---- digits ---------------------------------------------------------------------------------------------------------

// Digits of a value of a float16 or float32 layer.
__host__ __device__ constexpr int moe_digits(bool half) { return half ? 4 : 5; }

// v * 2^n, by two factors so that every n that occurs (below 2 * 126 in size) can be formed.
__device__ __forceinline__ float times_pow2(float v, int n) {
    const int a = n / 2;
    return v * __int_as_float((127 + a) << 23) * __int_as_float((127 + n - a) << 23);
}

// The shift s of a row whose largest magnitude has the bits `most`: v 2^s rounds to D balanced digits, the largest one's
// to nearly all their range. A row of zeros shifts by 0.
template <int D>
__device__ __forceinline__ int row_shift(uint32_t most) {
    if (most == 0) return 0;
    const int exponent = most >= 0x00800000u ? static_cast<int>(most >> 23) - 127 : -118 - __clz(most);
    const int s = 8 * D - 2 - exponent;  // the largest in [2^(8 D - 2), 2^(8 D - 1))
    const float limit = D == 4 ? 2139062016.0f : 547599876096.0f;  // 127 (256^D - 1) / 255, rounded down to a float32
    return times_pow2(__uint_as_float(most), s) > limit ? s - 1 : s;
}

constexpr int NOT_FINITE = 0x7FFF;  // in place of the shift of a row that holds an infinity or NaN

// What the sums over a row are to be shifted back by: they count units of the second lowest digit.
template <int D>
__device__ __forceinline__ int16_t shift_or_not(uint32_t most) {
    return static_cast<int16_t>(most < 0x7F800000u ? row_shift<D>(most) - 8 : NOT_FINITE);
}

// A digits' sum as the value it stands for.
__device__ __forceinline__ float shifted_back(long long sum, int shift) {
    return shift == NOT_FINITE ? NAN : times_pow2(__ll2float_rn(sum), -shift);
}

__device__ __forceinline__ bool finite_bits(uint32_t most) { return most < 0x7F800000u; }

// Four values of a row as D words of digits, the lowest digit first, at `to`, `to` + 128 ..
template <int D>
__device__ __forceinline__ void put_digits(const float4& v, int shift, uint8_t* to) {
    const float f[4] = {v.x, v.y, v.z, v.w};
    uint32_t word[D] = {};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        std::conditional_t<D == 5, long long, int> q;
        if constexpr (D == 5)
            q = __float2ll_rn(times_pow2(f[i], shift));
        else
            q = __float2int_rn(times_pow2(f[i], shift));
#pragma unroll
        for (int d = 0; d < D; d++) {
            const int digit = static_cast<int8_t>(q);
            word[d] |= static_cast<uint32_t>(digit & 0xFF) << (8 * i);
            q = (q - digit) >> 8;
        }
    }
#pragma unroll
    for (int d = 0; d < D; d++) *reinterpret_cast<uint32_t*>(to + d * moe::CHUNK) = word[d];
}

// Where value k (a multiple of 4) of a row chunk's digits lies. In step i of the chunk's four, lane q of a matrix column
// needs k = 32 i + 4 q .. and k = 32 i + 16 + 4 q ..; the words of steps 2 j and 2 j + 1 form its 16-byte unit (j, q), so
// that a column's four lanes read 64 consecutive bytes.
__device__ __forceinline__ int digit_place(int k) {
    return (k >> 6) * 64 + ((k >> 2) & 3) * 16 + ((k >> 5) & 1) * 8 + ((k >> 4) & 1) * 4;
}

__device__ __forceinline__ void moe_mma(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four bytes from byte `shift` / 8 of the word at addr on.
__device__ __forceinline__ uint32_t unaligned_word(uint32_t addr, uint32_t shift) {
    uint32_t lo, hi;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(lo) : "r"(addr) : "memory");
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(hi) : "r"(addr + 4) : "memory");
    return __funnelshift_r(lo, hi, shift);
}

// The 16 x 32 byte operand of one step: lane l gives the address of one of the four 8 x 16 byte parts' rows (rows 0-7 and
// 8-15 of the first 16 bytes, then of the second), every lane gets its four words in the order the instruction takes them.
__device__ __forceinline__ void load_rows(uint32_t (&a)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3])
                 : "r"(addr)
                 : "memory");
}

// ---- grid barrier ---------------------------------------------------------------------------------------------------

// The counts start every launch at zero. A CTA that gives up leaves without arriving any further, so a barrier that is
// passed has been reached by every CTA with its work done; the others' bounded waits at the next one run out too.

// Arrives and waits, bounded, for `target` arrivals; false when it gave up.
__device__ __forceinline__ bool grid_arrive(unsigned int* arrivals, unsigned int target, uint64_t limit_ns) {
    __threadfence();
    if (atomicAdd(arrivals, 1u) + 1u != target) {
        const uint64_t t0 = global_timer_ns();
        while (true) {
            unsigned int now;
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(now) : "l"(arrivals) : "memory");
            if (now >= target) break;
            if (global_timer_ns() - t0 > limit_ns) return false;
        }
    }
    __threadfence();
    return true;
}

// The whole CTA meets the grid for the time `which` (1 .. 4); false (for every thread) when this CTA has failed or gives up
// here. Out of line: the kernel runs each of its parts once or twice, so instructions that are fetched a second time are
// what it waits for.
static __device__ __noinline__ bool grid_barrier(unsigned int* arrivals, unsigned int which, uint64_t limit_ns,
                                                 const int* abort, int* failed) {
    __syncthreads();
    if (threadIdx.x == 0 && (*abort != 0 || !grid_arrive(arrivals, which * gridDim.x, limit_ns))) *failed = 1;
    __syncthreads();
    return *failed == 0;
}

// One thread of a CTA that is through with the counts (its last use of them, an acquiring load or fenced, comes before).
// The last one of the launch clears them for the next launch, whatever happened in this one.
__device__ __forceinline__ unsigned int count_out(const MoeLaunch& L) { return atomicAdd(&L.counts->exits, 1u); }

__device__ __forceinline__ void clear_counts(const MoeLaunch& L, unsigned int out_before) {
    if (out_before != gridDim.x - 1) return;
    __threadfence();
    *L.counts = MoeCounts{};
}

// A CTA that gives up raises the launch's failure.
__device__ __forceinline__ void leave_early(const MoeLaunch& L) {
    if (threadIdx.x != 0) return;
    atomicExch(L.error_flag, 1);
    __threadfence();
    clear_counts(L, count_out(L));
}

// The watchdog self-test: the second CTA comes late to the barrier `which`, later than the others wait.
static __device__ __noinline__ void come_late(uint64_t ns) {
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < ns) {
    }
}

__device__ __forceinline__ void self_test(const MoeLaunch& L, int which) {
    if (L.late_barrier == which && blockIdx.x == 1) come_late(L.late_ns);
}

// ---- phase 0 --------------------------------------------------------------------------------------------------------

__device__ __forceinline__ float moe_load(const void* p, int half, int64_t i) {
    return half ? __half2float(__ldg(static_cast<const __half*>(p) + i)) : __ldg(static_cast<const float*>(p) + i);
}

// Elements d .. d + 3 of a row of `size` that starts at element `row`, zeros past its end; VEC when they may be loaded as
// one (then size is a multiple of 4).
template <bool HALF, bool VEC>
__device__ __forceinline__ float4 moe_load4(const void* p, int64_t row, int d, int size) {
    const int64_t i = row + d;
    if constexpr (!VEC)
        return make_float4(d < size ? moe_load(p, HALF, i) : 0.0f, d + 1 < size ? moe_load(p, HALF, i + 1) : 0.0f,
                           d + 2 < size ? moe_load(p, HALF, i + 2) : 0.0f, d + 3 < size ? moe_load(p, HALF, i + 3) : 0.0f);
    if constexpr (!HALF) return __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + i));
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(static_cast<const __half*>(p) + i));
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    return make_float4(a.x, a.y, b.x, b.y);
}

// The start of part `part` of `total` things in `parts` nearly equal parts.
__device__ __forceinline__ int moe_split(int total, int part, int parts) {
    return static_cast<int>(static_cast<int64_t>(total) * part / parts);
}

// x as digits, row chunk by row chunk [D][128]. A warp finds its token's largest value and converts a part of four chunks.
template <class S, bool HALF, bool VEC>
__device__ __forceinline__ void moe_digits_x(const MoeFusedParams& p) {
    constexpr int D = moe_digits(HALF);
    const MoeLaunch& L = p.L;
    const int lane = threadIdx.x & 31;
    const int parts = (p.chunks_in + 3) / 4;
    // Spread over the CTAs, from the last one down: the first ones hold the router's units.
    for (int u = (threadIdx.x >> 5) * gridDim.x + gridDim.x - 1 - blockIdx.x; u < L.tokens * parts;
         u += gridDim.x * S::WARPS) {
        const int t = u / parts, part = u - t * parts;
        const int64_t x0 = static_cast<int64_t>(t) * L.model;
        const int vectors = (L.model + 3) / 4;
        uint32_t most = 0;
#pragma unroll 1
        for (int v0 = lane; v0 < vectors; v0 += 256) {
            float4 x[8];
#pragma unroll
            for (int i = 0; i < 8; i++)  // all in flight; past the end, the last vector again
                x[i] = moe_load4<HALF, VEC>(L.x, x0, 4 * min(v0 + 32 * i, vectors - 1), L.model);
#pragma unroll
            for (int i = 0; i < 8; i++)
                most = max(max(most, max(__float_as_uint(x[i].x) & 0x7FFFFFFFu, __float_as_uint(x[i].y) & 0x7FFFFFFFu)),
                           max(__float_as_uint(x[i].z) & 0x7FFFFFFFu, __float_as_uint(x[i].w) & 0x7FFFFFFFu));
        }
        most = __reduce_max_sync(0xFFFFFFFFu, most);
        if (part == 0 && lane == 0) L.x_most[t] = most;
        const int shift = finite_bits(most) ? row_shift<D>(most) : 0;
#pragma unroll 1
        for (int c = part * 4; c < min(part * 4 + 4, p.chunks_in); c++) {
            const int k = c * moe::CHUNK + lane * 4;
            const float4 x = k < L.model ? moe_load4<HALF, VEC>(L.x, x0, k, L.model) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            put_digits<D>(x, shift, L.x_digits + (static_cast<int64_t>(t) * p.chunks_in + c) * D * moe::CHUNK +
                                        digit_place(lane * 4));
        }
    }
    for (int i = blockIdx.x * S::THREADS + threadIdx.x; i < L.tokens * L.top_k; i += gridDim.x * S::THREADS)
        L.h_most[i] = 0;
}

// The hidden values as digits, in the same layout; zeros past the expert's size. A warp converts a chunk at a time.
template <class S, int D>
__device__ __forceinline__ void moe_digits_h(const MoeFusedParams& p) {
    const MoeLaunch& L = p.L;
    const int lane = threadIdx.x & 31;
    const int units = L.tokens * L.top_k * p.chunks_out;
#pragma unroll 1
    for (int u = (threadIdx.x >> 5) * gridDim.x + blockIdx.x; u < units; u += gridDim.x * S::WARPS) {
        const int pair = u / p.chunks_out, k = (u - pair * p.chunks_out) * moe::CHUNK + lane * 4;
        const uint32_t most = __ldcg(L.h_most + pair);
        float4 h = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (k < L.expert) h = __ldcg(reinterpret_cast<const float4*>(L.hidden + static_cast<int64_t>(pair) * p.hidden_pitch + k));
        if (k + 1 >= L.expert) h.y = 0.0f;  // the pitch's last elements are not written
        if (k + 2 >= L.expert) h.z = 0.0f;
        if (k + 3 >= L.expert) h.w = 0.0f;
        put_digits<D>(h, finite_bits(most) ? row_shift<D>(most) : 0,
                      L.h_digits + static_cast<int64_t>(u) * D * moe::CHUNK + digit_place(lane * 4));
    }
}

// Logits: units of one expert and 8 tokens, each shared by router_split warps of a CTA (so that a few units still occupy
// the SMs). Held in float64 from the products (exact there) to the ranking and the softmax: an error of float32's size in a
// large logit would be one of that size, not of its last bit, in a weight.
template <class S, bool HALF, bool VEC, bool ROUTER_HALF>
__device__ __forceinline__ void moe_logits(const MoeFusedParams& p, MoeShared<S>& sh) {
    const MoeLaunch& L = p.L;
    constexpr int TOKENS = S::MT == 1 ? 2 : 8;  // a unit has no more
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = p.router_split, per_cta = S::WARPS / split, part = warp % split;
    const int token_blocks = (L.tokens + 7) / 8, units = L.experts * token_blocks;
    const int vectors = (L.model + 3) / 4;  // of four elements; this warp's share of them
    const int v0 = moe_split(vectors, part, split), v1 = moe_split(vectors, part + 1, split);
    int buffer = 0;
    for (int first = blockIdx.x * per_cta; first < units; first += gridDim.x * per_cta, buffer ^= 1) {
        const int unit = first + warp / split;
        const int block = unit / L.experts, e = unit - block * L.experts, t0 = block * 8;  // a block's units lie together:
                                                                                          // blocks end on different CTAs
        const int n = unit < units ? min(8, L.tokens - t0) : 0;
        double sum[8];
#pragma unroll
        for (int i = 0; i < 8; i++) sum[i] = 0.0;
        if (n > 0) {
            const int64_t r0 = static_cast<int64_t>(e) * L.model, x0 = static_cast<int64_t>(t0) * L.model;
            // Past the tokens or the share, the last one again (its sums are dropped): every load of a step is in flight
            // at once.
            for (int v = v0 + lane; v < v1; v += 64) {
                float4 r[2], x[2][TOKENS];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int d = 4 * min(v + 32 * u, v1 - 1);
                    r[u] = moe_load4<ROUTER_HALF, VEC>(L.router, r0, d, L.model);
#pragma unroll
                    for (int i = 0; i < TOKENS; i++)
                        x[u][i] = moe_load4<HALF, VEC>(L.x, x0 + static_cast<int64_t>(min(i, n - 1)) * L.model, d, L.model);
                }
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    if (u == 1 && v + 32 >= v1) break;
                    const double rx = r[u].x, ry = r[u].y, rz = r[u].z, rw = r[u].w;
#pragma unroll
                    for (int i = 0; i < TOKENS; i++) {
                        sum[i] = fma(static_cast<double>(x[u][i].x), rx, sum[i]);
                        sum[i] = fma(static_cast<double>(x[u][i].y), ry, sum[i]);
                        sum[i] = fma(static_cast<double>(x[u][i].z), rz, sum[i]);
                        sum[i] = fma(static_cast<double>(x[u][i].w), rw, sum[i]);
                    }
                }
            }
        }
        // Lane bits 4, 3 and 2 choose the token: 4 + 2 + 1 exchanges, then two more within each token's four lanes.
        double a[4], b[2], c;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const double keep = lane & 16 ? sum[i + 4] : sum[i], give = lane & 16 ? sum[i] : sum[i + 4];
            a[i] = keep + __shfl_xor_sync(0xFFFFFFFFu, give, 16);
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const double keep = lane & 8 ? a[i + 2] : a[i], give = lane & 8 ? a[i] : a[i + 2];
            b[i] = keep + __shfl_xor_sync(0xFFFFFFFFu, give, 8);
        }
        c = (lane & 4 ? b[1] : b[0]) + __shfl_xor_sync(0xFFFFFFFFu, lane & 4 ? b[0] : b[1], 4);
        c += __shfl_xor_sync(0xFFFFFFFFu, c, 2);
        c += __shfl_xor_sync(0xFFFFFFFFu, c, 1);
        if ((lane & 3) == 0) sh.logit_part[buffer][warp][lane >> 2] = c;
        __syncthreads();
        if (part == 0 && lane < n) {
            double total = 0.0;
            for (int w = 0; w < split; w++) total += sh.logit_part[buffer][warp + w][lane];
            L.logits[static_cast<int64_t>(t0 + lane) * L.experts + e] = total;
        }
        if (L.tokens > S::WARPS && part == 0 && n > 0) {
            __syncwarp();
            if (lane == 0) {
                __threadfence();
                if (atomicAdd(&L.counts->tickets[t0 / 8], 1u) == static_cast<unsigned>(L.experts) - 1) atomicOr(&sh.complete, 1u << (t0 / 8));
            }
        }
    }
}

// ---- routing --------------------------------------------------------------------------------------------------------

// A key that orders numbers as unsigned ones; NaN below every number, with -infinity (what it ranks as).
__device__ __forceinline__ uint64_t rank_key(double v) {
    const uint64_t u = __double_as_longlong(isnan(v) ? -INFINITY : (v == 0.0 ? 0.0 : v));
    return u >> 63 ? ~u : u | uint64_t(1) << 63;  // -infinity is 0x000FFFFFFFFFFFFF: 0 marks a taken expert
}

__device__ __forceinline__ double rank_value(uint64_t key) {
    return __longlong_as_double(key >> 63 ? key & ~(uint64_t(1) << 63) : ~key);
}

// The largest key of a warp.
__device__ __forceinline__ uint64_t warp_max(uint64_t key) {
    const uint32_t high = __reduce_max_sync(0xFFFFFFFFu, static_cast<uint32_t>(key >> 32));
    const uint32_t low = __reduce_max_sync(0xFFFFFFFFu, static_cast<uint32_t>(key >> 32) == high ? static_cast<uint32_t>(key) : 0u);
    return static_cast<uint64_t>(high) << 32 | low;
}

// exp(d) for d <= 0 (or NaN) in float32, with what d's rounding to float32 drops.
__device__ __forceinline__ float exp_of(double d) {
    const float high = static_cast<float>(d);
    if (high < -150.0f) return 0.0f;  // below half the smallest float32
    const float e = expf(high);
    return fmaf(e, static_cast<float>(d - high), e);
}

// A token's experts by one warp: the largest key, the lowest expert among equals, top_k times. PER_LANE logits per lane.
template <class S, int D, int PER_LANE>
__device__ __forceinline__ void moe_choose(const MoeLaunch& L, MoeShared<S>& sh, int t, const double (&v)[PER_LANE],
                                           uint32_t x_most, bool publish) {
    const int lane = threadIdx.x & 31;
    uint64_t key[PER_LANE], best = 0;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < PER_LANE; i++) {
        key[i] = lane + 32 * i < L.experts ? rank_key(v[i]) : 0;
        nan |= lane + 32 * i < L.experts && isnan(v[i]);
        best = max(best, key[i]);
    }
    double top = rank_value(warp_max(best));
    if (__any_sync(0xFFFFFFFFu, nan)) top = NAN;  // the softmax of a row with a NaN is NaN
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < PER_LANE; i++)
        if (lane + 32 * i < L.experts) sum += exp_of(rank_value(key[i]) - top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    uint64_t picked = 0;  // lane k: the k-th expert's key and index
    int id = 0;
#pragma unroll 1
    for (int k = 0; k < L.top_k; k++) {
        uint64_t own = 0;
        int at = MOE_MAX_EXPERTS;
#pragma unroll
        for (int i = 0; i < PER_LANE; i++)
            if (key[i] > own) {
                own = key[i];
                at = lane + 32 * i;
            }
        const uint64_t most = warp_max(own);
        const int chosen_at = __reduce_min_sync(0xFFFFFFFFu, own == most ? at : MOE_MAX_EXPERTS);
        if (lane == k) {
            picked = most;
            id = chosen_at;
        }
#pragma unroll
        for (int i = 0; i < PER_LANE; i++)
            if (chosen_at == lane + 32 * i) key[i] = 0;
    }
    float weight = lane < L.top_k ? exp_of(rank_value(picked) - top) : 0.0f;
    float chosen = weight;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) chosen += __shfl_xor_sync(0xFFFFFFFFu, chosen, o);
    if (lane < L.top_k) {
        weight = weight / (L.normalize ? chosen : sum);
        const int i = t * L.top_k + lane;
        sh.id[i] = static_cast<uint16_t>(id);
        sh.weight[i] = weight;
        sh.shift[i] = shift_or_not<D>(x_most);
        if (publish) {
            L.ids[i] = id;
            L.weights[i] = weight;
            if (L.ids_out != nullptr) L.ids_out[i] = id;
            if (L.weights_out != nullptr) L.weights_out[i] = weight;
        }
    }
}

// Tokens first .. first + count - 1, a warp each.
template <class S, int D, int PER_LANE>
__device__ __forceinline__ void moe_choose_some(const MoeLaunch& L, MoeShared<S>& sh, int first, int count, bool publish) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll 1
    for (int t = first + warp; t < first + count; t += S::WARPS) {
        double v[PER_LANE];
#pragma unroll
        for (int i = 0; i < PER_LANE; i++)
            v[i] = lane + 32 * i < L.experts ? __ldcg(L.logits + static_cast<int64_t>(t) * L.experts + lane + 32 * i) : 0.0;
        moe_choose<S, D, PER_LANE>(L, sh, t, v, L.tokens > S::WARPS ? 0u : __ldcg(L.x_most + t), publish);
    }
}

template <class S, int D>
__device__ __forceinline__ void moe_choose_tokens(const MoeLaunch& L, MoeShared<S>& sh, int first, int count, bool publish) {
    if (L.experts <= 128)
        moe_choose_some<S, D, 4>(L, sh, first, count, publish);
    else
        moe_choose_some<S, D, MOE_MAX_EXPERTS / 32>(L, sh, first, count, publish);
}

// The pairs sorted by expert and cut into groups of at most 8 NT pairs; each thread lists its experts'. Within a group the
// pairs stand in the order the threads come in, which changes no result (a pair's sums do not depend on its column). Where
// an expert has more than one group, every CTA must cut its pairs alike: they are put in order first.
template <class S>
__device__ __forceinline__ void moe_group(const MoeLaunch& L, MoeShared<S>& sh) {
    constexpr int PER_THREAD = moe::MAX_PAIRS / S::THREADS, EXPERTS = MOE_MAX_EXPERTS / S::THREADS, FULL = 8 * S::NT;
    const int thread = threadIdx.x, warp = thread >> 5, lane = thread & 31;
    const int pairs = L.tokens * L.top_k;
#pragma unroll
    for (int i = 0; i < EXPERTS; i++) sh.count[thread * EXPERTS + i] = 0;
    __syncthreads();  // the choices are in, the counts are clear
    int rank[PER_THREAD];
#pragma unroll
    for (int i = 0; i < PER_THREAD; i++) {
        const int pair = thread + i * S::THREADS;
        if (pair >= pairs) break;
        rank[i] = atomicAdd(&sh.count[sh.id[pair]], 1);
    }
    __syncthreads();
    int count[EXPERTS], first = 0, group = 0;  // pairs; groups and, from bit 10 on, their units' cost (at most 768 and 40000)
    bool many = false;
#pragma unroll
    for (int i = 0; i < EXPERTS; i++) {
        count[i] = sh.count[thread * EXPERTS + i];
        first += count[i];
        group += (count[i] + FULL - 1) / FULL + (count[i] / FULL * unit_cost<S::NT>(FULL) << 10);
        if (count[i] % FULL != 0) group += unit_cost<S::NT>(count[i] % FULL) << 10;
        many |= count[i] > FULL;
    }
    if (__syncthreads_or(many)) {
#pragma unroll
        for (int i = 0; i < PER_THREAD; i++) {
            const int pair = thread + i * S::THREADS;
            if (pair >= pairs || sh.count[sh.id[pair]] <= FULL) continue;
            const uint32_t same = sh.id[pair];
            int less = 0;
#pragma unroll 1
            for (int j = 0; j < pair; j += 8) {  // ids past the pairs are never counted: they lie past `pair`
                const uint4 v = *reinterpret_cast<const uint4*>(&sh.id[j]);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    less += j + 2 * u < pair && (w[u] & 0xFFFFu) == same;
                    less += j + 2 * u + 1 < pair && (w[u] >> 16) == same;
                }
            }
            rank[i] = less;
        }
        __syncthreads();  // the counts have been read
    }
    const int own = first, own_groups = group;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {  // inclusive sums over the experts
        const int a = __shfl_up_sync(0xFFFFFFFFu, first, o), b = __shfl_up_sync(0xFFFFFFFFu, group, o);
        if (lane >= o) {
            first += a;
            group += b;
        }
    }
    if (lane == 31) {
        sh.warp_total[0][warp] = first;
        sh.warp_total[1][warp] = group;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < S::WARPS; w++)
        if (w < warp) {
            first += sh.warp_total[0][w];
            group += sh.warp_total[1][w];
        }
    if (thread == S::THREADS - 1) {
        sh.groups = group & 1023;
        sh.cost = group >> 10;
    }
    first -= own;
    group -= own_groups;
    int cost = group >> 10;
    group &= 1023;
#pragma unroll
    for (int i = 0; i < EXPERTS; i++) {
        const int e = thread * EXPERTS + i;
        sh.count[e] = first;
        for (int done = 0; done < count[i]; done += FULL) {
            const int n = min(FULL, count[i] - done);
            sh.group[group++] = MoeGroup{static_cast<uint16_t>(e), static_cast<uint16_t>(first + done),
                                         static_cast<uint16_t>(n), static_cast<uint16_t>(cost)};
            cost += unit_cost<S::NT>(n);
        }
        first += count[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER_THREAD; i++) {
        const int pair = thread + i * S::THREADS;
        if (pair >= pairs) break;
        sh.order[sh.count[sh.id[pair]] + rank[i]] = static_cast<uint16_t>(pair);
    }
    __syncthreads();
}

// ---- phases 1 and 2 -------------------------------------------------------------------------------------------------

// One phase's work of this warp. The CTA owns units [u0, u0 + units). Its warps take whole units in turn, walking K
// together, so that they find the columns' digits in L1; the units left over after the full rounds go to a warp each if
// there are many, and are otherwise cut into equal runs of chunks, so that every warp keeps boxes in flight to the end.
// Position i of a warp's work: chunk i % chunks of its unit i / chunks for i < rounds * chunks, then the run
// [at, end) of the chunks of units u0 + tail ..
struct MoeRange {
    int u0, units;
    int rounds;   // whole units of this warp
    int tail;     // units before the cut ones
    int at, end;  // the warp's run of the cut units' chunks
};

// Where the share of CTA `block` starts: a group, and how far into its units (a fraction of 2^16). Shares cost the same.
struct MoePlace {
    int group;
    uint32_t into;
    __device__ __forceinline__ int unit(int blocks) const {
        return group * blocks + static_cast<int>((static_cast<uint64_t>(into) * blocks) >> 16);
    }
};

template <class S>
__device__ __forceinline__ MoePlace moe_place(const MoeShared<S>& sh, unsigned block) {
    const unsigned scaled = static_cast<unsigned>(sh.cost) * block, whole = scaled / gridDim.x;  // below 2^16 * 2^10
    const unsigned part = ((scaled - whole * gridDim.x) << 16) / gridDim.x;
    int low = 0, high = sh.groups;  // the last group that does not start past it
    while (high - low > 1) {
        const int mid = (low + high) / 2;
        if (sh.group[mid].before <= whole)
            low = mid;
        else
            high = mid;
    }
    const MoeGroup& g = sh.group[low];
    return {low, ((whole - g.before) << 16 | part) / static_cast<unsigned>(unit_cost<S::NT>(g.count))};
}

template <class S>
__device__ __forceinline__ MoeRange moe_range(int first, int past, int chunks, int warp) {
    MoeRange r;
    r.u0 = first;
    r.units = past - first;
    r.rounds = r.units / S::WARPS;
    r.tail = r.rounds * S::WARPS;
    int left = r.units - r.tail;
    if (left >= S::WHOLE_FROM) {
        r.rounds += warp < left;
        r.tail = r.units;
        left = 0;
    }
    r.at = moe_split(left * chunks, warp, S::WARPS);
    r.end = moe_split(left * chunks, warp + 1, S::WARPS);
    return r;
}

// The warp that holds chunk i of `total`.
template <class S>
__device__ __forceinline__ int moe_owner(int i, int total) {
    return static_cast<int>((static_cast<int64_t>(i + 1) * S::WARPS - 1) / total);
}

// Out of line for the same reason as grid_barrier: eight copies of five activations took 162 us (64 tokens through 6 of 64
// experts) where this takes 154.
static __device__ __noinline__ float moe_activate(float v, int kind) {
    float f[1] = {v};
    activate_all(f, kind);
    return f[0];
}

// What the warp's ring loads next: phase 1's work, then phase 2's.
struct MoeFeed {
    int phase;
    int rounds;        // whole units still to begin
    int unit;          // the unit being loaded
    int left;          // boxes left of this run of boxes (a unit, or the run over the cut units)
    int x, x_end;      // byte of K of the next box, and past the last one
    int y, e;          // row and expert (gate half) of the next box
    bool whole;        // a whole unit, walked around from its first box
    uint32_t issued;   // boxes so far
};

template <class S, int D>
struct MoeWarp {
    static constexpr int NT = S::NT, MT = S::MT;
    const MoeFusedParams& p;
    MoeShared<S>& sh;
    const CUtensorMap* map_in;
    const CUtensorMap* map_out;
    uint8_t* ring;
    uint64_t* full;
    int warp, lane;
    MoeRange range_in, range_out;
    MoeFeed feed;
    uint32_t taken;  // boxes read so far
    float2 scale[MT];  // of the unit at hand

    // Whole units are walked around from a chunk that differs from CTA to CTA: in step, all CTAs would read the same few
    // columns of rows a power of two apart (8 tokens through 2 of 2 experts, 4096 x 8192: phase 1 33.3 us in step, 26.9 so).
    __device__ __forceinline__ static int first_chunk(int chunks) {
        return MT == 1 ? 0 : static_cast<int>(static_cast<unsigned>(chunks) * blockIdx.x / gridDim.x);
    }

    __device__ __forceinline__ int chunks(int phase) const { return phase == 0 ? p.chunks_in : p.chunks_out; }
    __device__ __forceinline__ int blocks(int phase) const { return phase == 0 ? p.blocks_in : p.blocks_out; }

    // Points the feed at a unit of its phase.
    __device__ __forceinline__ void aim(int unit) {
        const int b = blocks(feed.phase), group = unit / b;
        const bool halves = feed.phase == 0 && p.L.gated;
        feed.unit = unit;
        feed.y = (unit - group * b) * (halves ? 8 * MT : 16 * MT);
        feed.e = sh.group[group].expert * (halves ? 2 : 1);
    }

    // The next run of boxes; false when there is none.
    __device__ __forceinline__ bool next_run() {
        while (true) {
            const MoeRange& r = feed.phase == 0 ? range_in : range_out;
            const int c = chunks(feed.phase);
            if (feed.rounds < r.rounds) {
                aim(r.u0 + feed.rounds * S::WARPS + warp);
                feed.x = first_chunk(c) * moe::CHUNK;
                feed.x_end = c * moe::CHUNK;
                feed.whole = true;
                feed.left = c;
                feed.rounds++;
                return true;
            }
            if (feed.rounds == r.rounds && r.at < r.end) {
                feed.rounds++;
                const int local = r.at / c;
                aim(r.u0 + r.tail + local);
                feed.x = (r.at - local * c) * moe::CHUNK;
                feed.x_end = c * moe::CHUNK;
                feed.left = r.end - r.at;
                feed.whole = false;
                return true;
            }
            if (feed.phase == 1) return false;
            feed.phase = 1;
            feed.rounds = 0;
        }
    }

    // Row r of a box, as a row of the weights' matrix of its phase: rows past the expert's size are its last one again (their
    // sums are not stored).
    __device__ __forceinline__ int64_t weight_row(int phase, int e, int y, int r) const {
        const bool halves = phase == 0 && p.L.gated;
        const int size = phase == 0 ? p.L.expert : p.L.model;
        const int half = halves && r >= 8 * MT ? 1 : 0;
        return (static_cast<int64_t>(e) + half) * size + min(y + r - half * 8 * MT, size - 1);
    }

    // The aligned 16-byte units around the feed's 128 bytes of each row, nine a row, copied asynchronously; zeros for those
    // that start past the weights.
    __device__ __forceinline__ void copy_rows(uint8_t* box) const {
        const int8_t* w = feed.phase == 0 ? p.L.w_in : p.L.w_out;
        const int8_t* end = feed.phase == 0 ? p.end_in : p.end_out;
        const int ld = feed.phase == 0 ? p.L.model : p.L.expert;
        constexpr int UNITS = S::ROWS * 9;
#pragma unroll 3
        for (int u0 = 0; u0 < UNITS; u0 += 32) {
            const int u = u0 + lane;
            if (u >= UNITS) break;
            const int r = u / 9, j = u - 9 * r;
            const uintptr_t at = reinterpret_cast<uintptr_t>(w + weight_row(feed.phase, feed.e, feed.y, r) * ld + feed.x);
            const int8_t* src = reinterpret_cast<const int8_t*>((at & ~uintptr_t(15)) + 16 * j);
            const bool ok = src < end;  // else nothing is read; the address is one that is read elsewhere
            const int8_t* from = ok ? src : reinterpret_cast<const int8_t*>(reinterpret_cast<uintptr_t>(w) & ~uintptr_t(15));
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(box + r * S::PITCH + 16 * j)),
                         "l"(from), "r"(ok ? 16 : 0)
                         : "memory");
        }
    }

    // Issues the next box if any is left; the caller has freed a slot.
    __device__ __forceinline__ void issue() {
        if (feed.left == 0 && !next_run()) {
            if constexpr (!S::ALIGNED) cp_async_commit();  // an empty group keeps their count
            return;
        }
        const int slot = feed.issued % moe::SLOTS;
        if constexpr (S::ALIGNED) {
            if (lane == 0) {
                mbar_arrive_expect_tx(&full[slot], S::BOX);
                tma_load_3d(ring + slot * S::BOX, feed.phase == 0 ? map_in : map_out, &full[slot], feed.x, feed.y, feed.e);
            }
        } else {
            copy_rows(ring + slot * S::BOX);
            cp_async_commit();
        }
        feed.issued++;
        feed.left--;
        feed.x += moe::CHUNK;
        if (feed.x == feed.x_end && feed.left > 0) {
            feed.x = 0;
            if (!feed.whole) aim(feed.unit + 1);
        }
    }

    // The digits of n-tile t's columns in one chunk: v points at the chunk of row 0 (this lane's 16 bytes).
    __device__ __forceinline__ static void load_digits(uint4 (&b)[D][2], const uint8_t* v) {
#pragma unroll
        for (int d = 0; d < D; d++)
#pragma unroll
            for (int j = 0; j < 2; j++) b[d][j] = *reinterpret_cast<const uint4*>(v + d * moe::CHUNK + j * 64);
    }

    // The digits' sums of one unit's chunks [c0, c1): rows g and g + 8 of matrix tile i, columns 2 q and 2 q + 1 of n-tile
    // t in acc[i][t][digit - 1]. The columns' digits start at values + row[t] (column g of the tile). `halves`: the box holds
    // the gate's rows, then the other half's, and a tile 8 of each.
    __device__ __forceinline__ bool products(const uint8_t* values, const uint32_t (&row)[NT], int tiles, bool halves,
                                             const uint32_t (&skew)[MT][2], int c0, int count, int wrap,
                                             int (&acc)[MT][NT][D - 1][4]) {
        // Where registers allow, the next chunk's digits of tile 0 are on their way while one is multiplied (64 tokens through
        // 6 of 64 experts 172 -> 165 us); elsewhere they are asked for before the wait for the box. The other tiles' are when
        // their turn comes.
        constexpr bool AHEAD = MT == 2 && NT * (D - 1) <= 12;
        const int q = lane & 3;
        // This lane's row of the parts of a step: part lane / 8 is rows 0-7 or 8-15 (odd) of the first or second (2, 3)
        // 16 bytes. A box's 16-byte units are swizzled by the row (its low three bits are lane % 8 in every part), so eight
        // lanes of a part touch eight different units of 128 bytes: no bank conflict.
        const int tile_step = (halves ? 8 : 16) * S::PITCH, half_step = (halves ? 8 * MT : 8) * S::PITCH;
        const uint32_t my_row = smem_u32(ring) + (lane & 7) * moe::CHUNK + ((lane >> 3) & 1) * half_step;
        const uint32_t my_unit = lane >> 4, my_swizzle = lane & 7;
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int d = 0; d < D - 1; d++)
#pragma unroll
                    for (int i = 0; i < 4; i++) acc[m][t][d][i] = 0;
        const uint8_t* v = values + c0 * D * moe::CHUNK + q * 16;
        uint4 next[D][2];
        if constexpr (AHEAD) load_digits(next, v + row[0]);
#pragma unroll 1
        for (int c = c0; count > 0; count--) {
            const uint8_t* here = v;
            if (++c == wrap) {
                c = 0;
                v = values + q * 16;
            } else {
                v += D * moe::CHUNK;
            }
            const int slot = taken % moe::SLOTS;
            uint4 b[D][2];
            if constexpr (AHEAD) {
#pragma unroll
                for (int d = 0; d < D; d++)
#pragma unroll
                    for (int j = 0; j < 2; j++) b[d][j] = next[d][j];
                if (count > 1) load_digits(next, v + row[0]);
            } else {
                load_digits(b, here + row[0]);
            }
            uint32_t a[MT][4][4];
            if constexpr (S::ALIGNED) {
                const bool ok = mbar_wait(&full[slot], (taken / moe::SLOTS) & 1, &sh.abort);
                if (!__all_sync(0xFFFFFFFFu, ok)) return false;
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        load_rows(a[m][i], my_row + slot * S::BOX + m * tile_step + (((2 * i + my_unit) ^ my_swizzle) << 4));
            } else {
                cp_async_wait_group<moe::SLOTS - 1>();  // the oldest of the copies
                __syncwarp();
                // Bytes 32 i + 4 q (+ 16) of rows g and g + 8, which start `skew` bytes into their units: the rows lie
                // 36 words apart, so equal skews meet no bank conflict.
                const uint32_t box = smem_u32(ring) + slot * S::BOX + (lane >> 2) * S::PITCH + q * 4;
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const uint32_t at = box + m * tile_step + h * half_step + (skew[m][h] & ~3u);
                        const uint32_t shift = (skew[m][h] & 3u) * 8;
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            a[m][i][h] = unaligned_word(at + 32 * i, shift);
                            a[m][i][2 + h] = unaligned_word(at + 32 * i + 16, shift);
                        }
                    }
            }
            taken++;
#pragma unroll
            for (int t = 0; t < NT; t++) {
                if (t >= tiles) break;
                if (t > 0) load_digits(b, here + row[t]);
                int low[MT][4] = {};
#pragma unroll
                for (int j = 0; j < 2; j++) {
#pragma unroll
                    for (int m = 0; m < MT; m++) moe_mma(low[m], a[m][2 * j], b[0][j].x, b[0][j].y);
#pragma unroll
                    for (int m = 0; m < MT; m++)
#pragma unroll
                        for (int d = 1; d < D; d++) moe_mma(acc[m][t][d - 1], a[m][2 * j], b[d][j].x, b[d][j].y);
#pragma unroll
                    for (int m = 0; m < MT; m++) moe_mma(low[m], a[m][2 * j + 1], b[0][j].z, b[0][j].w);
#pragma unroll
                    for (int m = 0; m < MT; m++)
#pragma unroll
                        for (int d = 1; d < D; d++) moe_mma(acc[m][t][d - 1], a[m][2 * j + 1], b[d][j].z, b[d][j].w);
                }
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int i = 0; i < 4; i++) acc[m][t][0][i] += (low[m][i] + 128) >> 8;  // at most 2^21 in size before
                // Every row part has been an operand, so the slot's reads are done: a box loaded over it any earlier could
                // overtake reads that still wait in line behind the digits' loads.
                if (t == 0) {
                    __syncwarp();
                    issue();
                }
            }
        }
        return true;
    }

    // The digits' sums as one, exact in units of the second lowest digit.
    __device__ __forceinline__ static long long whole(const int (&acc)[D - 1][4], int i) {
        long long sum = acc[D - 2][i];
#pragma unroll
        for (int d = D - 3; d >= 0; d--) sum = sum * 256 + acc[d][i];
        return sum;
    }

    // The scales of rows g and g + 8 of a unit's tiles. Asked for before its products and (volatile) not later: behind the
    // weights queued in DRAM such a load takes some 3 us.
    __device__ __forceinline__ void scales(int phase, const MoeGroup& grp, int block) {
        const MoeLaunch& L = p.L;
        const bool halves = phase == 0 && L.gated;
        const int size = phase == 0 ? L.expert : L.model;
        const int other = halves ? size : 8;
        const float* s = (phase == 0 ? L.in_scale : L.out_scale) + static_cast<int64_t>(grp.expert) * (halves ? 2 : 1) * size;
#pragma unroll
        for (int m = 0; m < MT; m++) {
            const int r = (block * MT + m) * (halves ? 8 : 16) + (lane >> 2);
            scale[m] = make_float2(0.0f, 0.0f);
            if (r < size) asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(scale[m].x) : "l"(s + r));
            if (halves ? r < size : r + 8 < size) asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(scale[m].y) : "l"(s + r + other));
        }
    }

    // Phase 1's results: the hidden values and each pair's largest.
    __device__ __forceinline__ void finish_in(const MoeGroup& grp, int block, const long long (&sum)[MT][NT][4]) {
        const MoeLaunch& L = p.L;
        const int g = lane >> 2, q = lane & 3;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            if (8 * t >= grp.count) break;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int n = 8 * t + 2 * q + i;
                const int pair = sh.order[grp.first + min(n, grp.count - 1)];
                const int shift = sh.shift[pair];
                float* hidden = L.hidden + static_cast<int64_t>(pair) * p.hidden_pitch;
                uint32_t most = 0;
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    const int j0 = (block * MT + m) * (L.gated ? 8 : 16) + g;
                    float h[2] = {shifted_back(sum[m][t][i], shift) * scale[m].x,
                                  shifted_back(sum[m][t][2 + i], shift) * scale[m].y};
                    if (L.gated) {
                        h[0] = moe_activate(h[0], L.activation) * h[1];
                    } else {
                        h[0] = moe_activate(h[0], L.activation);
                        h[1] = moe_activate(h[1], L.activation);
                        if (n < grp.count && j0 + 8 < L.expert) {
                            hidden[j0 + 8] = h[1];
                            most = max(most, __float_as_uint(h[1]) & 0x7FFFFFFFu);
                        }
                    }
                    if (n < grp.count && j0 < L.expert) {
                        hidden[j0] = h[0];
                        most = max(most, __float_as_uint(h[0]) & 0x7FFFFFFFu);
                    }
                }
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
                if (g == 0 && n < grp.count) atomicMax(&sh.most[pair], most);
            }
        }
    }

    // Phase 2's results: the pair's weight times the row's scale times the sum.
    __device__ __forceinline__ void finish_out(const MoeGroup& grp, int block, const long long (&sum)[MT][NT][4]) {
        const MoeLaunch& L = p.L;
        const int g = lane >> 2, q = lane & 3;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            if (8 * t >= grp.count) break;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int n = 8 * t + 2 * q + i;
                if (n >= grp.count) continue;
                const int pair = sh.order[grp.first + n];
                const int shift = sh.shift[pair];
                const float weight = sh.weight[pair];
                float* to = L.outputs + static_cast<int64_t>(pair) * p.out_pitch;
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    const int d0 = (block * MT + m) * 16 + g;
                    if (d0 < L.model) to[d0] = weight * (shifted_back(sum[m][t][i], shift) * scale[m].x);
                    if (d0 + 8 < L.model) to[d0 + 8] = weight * (shifted_back(sum[m][t][2 + i], shift) * scale[m].y);
                }
            }
        }
    }

    __device__ __forceinline__ long long* segment(int warp, int which) const {
        return p.L.segments + (static_cast<int64_t>(blockIdx.x * S::WARPS + warp) * 2 + which) * S::SUMS;
    }

    // The warp's range of one phase. False (for the whole CTA) when a wait gave up.
    __device__ __forceinline__ bool run(int phase) {
        const MoeRange r = phase == 0 ? range_in : range_out;
        const int c = chunks(phase), per_group = blocks(phase), total = (r.units - r.tail) * c;
        const uint8_t* values = phase == 0 ? p.L.x_digits : p.L.h_digits;
        const uint32_t row_bytes = static_cast<uint32_t>(c) * D * moe::CHUNK;
        const int g = lane >> 2;
        // The unit that this warp's run cuts at its end, if the run holds its start: finished after the others.
        int local = (r.end - 1) / c;
        const int cut = r.at < r.end && local * c >= r.at && local * c + c > r.end ? local : -1;
        int round = 0, at = r.at;
        bool last_pass = false;
#pragma unroll 1
        while (true) {
            // A pass: a segment of a unit (its sums, to be finished or left in `segments`), then, once all warps are
            // through theirs, the cut unit.
            int c0 = 0, c1 = c, unit;
            const bool in_round = round < r.rounds;
            if (in_round) {
                unit = r.u0 + round * S::WARPS + warp;
            } else if (at < r.end) {
                local = at / c;
                c0 = at - local * c;
                c1 = min(c, c0 + r.end - at);
                unit = r.u0 + r.tail + local;
            } else {
                if (last_pass) break;
                last_pass = true;
                __syncthreads();
                if (sh.abort || cut < 0) break;
                unit = r.u0 + r.tail + cut;
            }
            const int group = unit / per_group, block = unit - group * per_group;
            const MoeGroup grp = sh.group[group];
            const int tiles = (grp.count + 7) / 8;
            const bool is_whole = c1 - c0 == c;
            if (!last_pass && (is_whole || (!in_round && local == cut))) scales(phase, grp, block);  // a cut one's is kept
            long long sum[MT][NT][4];
            if (!last_pass) {
                uint32_t row[NT];
#pragma unroll
                for (int t = 0; t < NT; t++) {  // columns past the group's pairs repeat its last one and are not stored
                    const int pair = sh.order[grp.first + min(8 * t + g, grp.count - 1)];
                    row[t] = static_cast<uint32_t>(phase == 0 ? pair / p.L.top_k : pair) * row_bytes;
                }
                int acc[MT][NT][D - 1][4];
                const bool halves = phase == 0 && p.L.gated;
                uint32_t skew[MT][2] = {};
                if constexpr (!S::ALIGNED) {
                    const int8_t* w = phase == 0 ? p.L.w_in : p.L.w_out;
                    const int ld = phase == 0 ? p.L.model : p.L.expert;
#pragma unroll
                    for (int m = 0; m < MT; m++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const int r = m * (halves ? 8 : 16) + h * (halves ? 8 * MT : 8) + g;
                            const int64_t at = weight_row(phase, grp.expert * (halves ? 2 : 1), block * (halves ? 8 * MT : 16 * MT), r) * ld;
                            skew[m][h] = static_cast<uint32_t>((reinterpret_cast<uintptr_t>(w) + at) & 15);
                        }
                }
                if (!products(values, row, tiles, halves, skew, in_round ? first_chunk(c) : c0, c1 - c0, c, acc)) {  // the abort flag is up
                    round = r.rounds;
                    at = r.end;
                    continue;
                }
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++) sum[m][t][i] = whole(acc[m][t], i);
                if (!is_whole) {
                    longlong2* to = reinterpret_cast<longlong2*>(segment(warp, at == r.at ? 0 : 1)) + lane;
#pragma unroll
                    for (int t = 0; t < NT; t++)
                        if (t < tiles) {
#pragma unroll
                            for (int m = 0; m < MT; m++) {
                                to[64 * (MT * t + m)] = make_longlong2(sum[m][t][0], sum[m][t][1]);
                                to[64 * (MT * t + m) + 32] = make_longlong2(sum[m][t][2], sum[m][t][3]);
                            }
                        }
                }
                if (in_round)
                    round++;
                else
                    at += c1 - c0;
                if (!is_whole) continue;
            } else {
                // Its own segment is its last one (or, starting at its range's start, its first), the others' their first.
                const int i0 = cut * c, last = moe_owner<S>(i0 + c - 1, total);
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++) sum[m][t][i] = 0;
#pragma unroll 1
                for (int w = warp; w <= last; w++) {
                    if (moe_split(total, w, S::WARPS) == moe_split(total, w + 1, S::WARPS)) continue;  // no share
                    const longlong2* from =
                        reinterpret_cast<const longlong2*>(segment(w, w == warp && i0 != r.at ? 1 : 0)) + lane;
#pragma unroll
                    for (int t = 0; t < NT; t++)
                        if (t < tiles) {
#pragma unroll
                            for (int m = 0; m < MT; m++) {
                                const longlong2 u = from[64 * (MT * t + m)], v = from[64 * (MT * t + m) + 32];
                                sum[m][t][0] += u.x;
                                sum[m][t][1] += u.y;
                                sum[m][t][2] += v.x;
                                sum[m][t][3] += v.y;
                            }
                        }
                }
            }
            if (phase == 0)
                finish_in(grp, block, sum);
            else
                finish_out(grp, block, sum);
        }
        return sh.abort == 0;
    }

    // Waits (bounded) for boxes still in flight: none may land after the CTA has gone.
    __device__ __forceinline__ void drain() {
        if constexpr (!S::ALIGNED) {
            cp_async_wait_all();
            return;
        }
        int give_up = 0;
        while (taken != feed.issued) {
            if (!mbar_wait(&full[taken % moe::SLOTS], (taken / moe::SLOTS) & 1, &give_up)) break;
            taken++;
        }
    }
};

template <bool HALF, class S>
__global__ void __launch_bounds__(S::THREADS, 1)
    moe_fused_kernel(const __grid_constant__ CUtensorMap map_in, const __grid_constant__ CUtensorMap map_out,
                     const __grid_constant__ MoeFusedParams p) {
    constexpr int D = moe_digits(HALF);
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    MoeShared<S>& sh = *reinterpret_cast<MoeShared<S>*>(smem + S::RING);
    const MoeLaunch& L = p.L;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_trigger();
    if (threadIdx.x == 0) {
        for (int w = 0; w < S::WARPS; w++)
            for (int s = 0; s < moe::SLOTS; s++) mbar_init(&sh.full[w][s], 1);
        sh.abort = 0;
        sh.failed = 0;
        sh.complete = 0;
        fence_mbar_init();
        if constexpr (S::ALIGNED) {
            prefetch_tmap(&map_in);
            prefetch_tmap(&map_out);
        }
    }
    pdl_wait();
    self_test(L, 1);
    for (int i = threadIdx.x; i < L.tokens * L.top_k; i += S::THREADS) sh.most[i] = 0;
    if (p.vec)
        moe_digits_x<S, HALF, true>(p);
    else
        moe_digits_x<S, HALF, false>(p);
    if (!p.vec)
        L.router_half ? moe_logits<S, HALF, false, true>(p, sh) : moe_logits<S, HALF, false, false>(p, sh);
    else
        L.router_half ? moe_logits<S, HALF, true, true>(p, sh) : moe_logits<S, HALF, true, false>(p, sh);
    if (L.tokens > S::WARPS) {
        __syncthreads();
        __threadfence();  // the other CTAs' logits of the blocks completed here
        for (unsigned left = sh.complete; left != 0; left &= left - 1) {
            const int t0 = 8 * (__ffs(left) - 1);
            moe_choose_tokens<S, D>(L, sh, t0, min(8, L.tokens - t0), true);
        }
    }
    auto meet = [&](unsigned int which) {
        return grid_barrier(&L.counts->arrivals, which, L.wait_limit_ns, &sh.abort, &sh.failed);
    };
    if (!meet(1)) {
        leave_early(L);
        return;
    }
    if (L.tokens <= S::WARPS) {
        moe_choose_tokens<S, D>(L, sh, 0, L.tokens, blockIdx.x == 0);
    } else {
        for (int i = threadIdx.x; i < L.tokens * L.top_k; i += S::THREADS) {
            sh.id[i] = static_cast<uint16_t>(__ldcg(L.ids + i));
            sh.weight[i] = __ldcg(L.weights + i);
            sh.shift[i] = shift_or_not<D>(__ldcg(L.x_most + i / L.top_k));
        }
    }
    moe_group(L, sh);

    MoeWarp<S, D> me{p, sh, &map_in, &map_out, smem + warp * moe::SLOTS * S::BOX, sh.full[warp], warp, lane, {}, {}, {}, 0, {}};
    if constexpr (S::MT == 1) {  // one or two tokens: every unit costs the same
        const int units_in = sh.groups * p.blocks_in, units_out = sh.groups * p.blocks_out;
        me.range_in = moe_range<S>(moe_split(units_in, blockIdx.x, gridDim.x), moe_split(units_in, blockIdx.x + 1, gridDim.x),
                                   p.chunks_in, warp);
        me.range_out = moe_range<S>(moe_split(units_out, blockIdx.x, gridDim.x),
                                    moe_split(units_out, blockIdx.x + 1, gridDim.x), p.chunks_out, warp);
    } else {
        const MoePlace mine = moe_place(sh, blockIdx.x + (lane & 1));  // even lanes: the share's start, odd ones: its end
        auto of = [&](int l) {
            return MoePlace{__shfl_sync(0xFFFFFFFFu, mine.group, l), __shfl_sync(0xFFFFFFFFu, mine.into, l)};
        };
        const MoePlace from = of(0), to = of(1);
        me.range_in = moe_range<S>(from.unit(p.blocks_in), to.unit(p.blocks_in), p.chunks_in, warp);
        me.range_out = moe_range<S>(from.unit(p.blocks_out), to.unit(p.blocks_out), p.chunks_out, warp);
    }
    for (int s = 0; s < moe::SLOTS; s++) me.issue();

#pragma unroll 1
    for (int phase = 0; phase < 2; phase++) {
        const bool ok = me.run(phase);
        if (phase == 1) break;
        if (ok) {
            __syncthreads();  // every warp's largest values are in
            for (int i = threadIdx.x; i < L.tokens * L.top_k; i += S::THREADS)
                if (sh.most[i] != 0) atomicMax(L.h_most + i, sh.most[i]);
        }
        self_test(L, 2);
        if (!meet(2)) {
            me.drain();
            leave_early(L);
            return;
        }
        moe_digits_h<S, D>(p);
        self_test(L, 3);
        if (!meet(3)) {
            me.drain();
            leave_early(L);
            return;
        }
        for (int i = threadIdx.x; i < L.tokens * L.top_k; i += S::THREADS)
            sh.shift[i] = shift_or_not<D>(__ldcg(L.h_most + i));
        __syncthreads();
    }
    me.drain();
    self_test(L, 4);
    if (!meet(4)) {
        leave_early(L);
        return;
    }
    const unsigned int out_before = threadIdx.x == 0 ? count_out(L) : 0;  // its answer comes while the sums are formed
    const int vectors = (L.model + 3) / 4, total = L.tokens * vectors;
    for (int i = blockIdx.x * S::THREADS + threadIdx.x; i < total; i += gridDim.x * S::THREADS) {
        const int t = i / vectors, d = (i - t * vectors) * 4;
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int k = 0; k < L.top_k; k++) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(
                L.outputs + (static_cast<int64_t>(t) * L.top_k + k) * p.out_pitch + d));
            sum.x += v.x;
            sum.y += v.y;
            sum.z += v.z;
            sum.w += v.w;
        }
        const float out[4] = {sum.x, sum.y, sum.z, sum.w};
        const int64_t at = static_cast<int64_t>(t) * L.model + d;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            if (d + u >= L.model) break;
            if constexpr (HALF) {
                const float r = L.residual != nullptr ? __half2float(static_cast<const __half*>(L.residual)[at + u]) : 0.0f;
                static_cast<__half*>(L.y)[at + u] = __float2half_rn(out[u] + r);
            } else {
                const float r = L.residual != nullptr ? static_cast<const float*>(L.residual)[at + u] : 0.0f;
                static_cast<float*>(L.y)[at + u] = out[u] + r;
            }
        }
    }
    if (threadIdx.x == 0) clear_counts(L, out_before);
}

// ---- host side ------------------------------------------------------------------------------------------------------

// The shape of a launch: NT and MT.
struct MoeChoice {
    int nt, mt, warps;
};

// Groups of 8 columns hold all of an expert's tokens up to 8 tokens; groups of 16 most of them while the experts see 10
// on average at most.
static MoeChoice moe_choice(const MoeLaunch& L) {
    if (L.tokens <= 2) return {1, 1, moe::Shape<1, 1, true>::WARPS};
    const int nt = L.tokens <= 8 ? 1 : L.tokens * L.top_k <= 10 * L.experts ? 2 : 4;
    return {nt, 2, moe::Shape<1, 2, true>::WARPS};
}

static int chunks_of(int size) { return (size + moe::CHUNK - 1) / moe::CHUNK; }

bool moe_aligned(const MoeLaunch& L) {
    auto aligned = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
    return L.model % 16 == 0 && L.expert % 16 == 0 && aligned(L.w_in) && aligned(L.w_out);
}

static int round4(int v) { return (v + 3) & ~3; }

MoeFusedSizes moe_fused_sizes(const MoeLaunch& L) {
    const int64_t pairs = int64_t(L.tokens) * L.top_k;
    MoeFusedSizes s;
    s.logits = int64_t(L.tokens) * L.experts * 8;
    const int digits = moe_digits(L.x_half);
    s.x_digits = int64_t(L.tokens) * chunks_of(L.model) * digits * moe::CHUNK;
    s.h_digits = pairs * chunks_of(L.expert) * digits * moe::CHUNK;
    s.x_most = int64_t(L.tokens) * 4;
    s.h_most = pairs * 4;
    s.outputs = pairs * round4(L.model) * 4;
    s.hidden = pairs * round4(L.expert) * 4;
    const MoeChoice shape = moe_choice(L);
    s.segments = int64_t(L.num_sms) * shape.warps * 2 * (16 * shape.mt) * (8 * shape.nt) * int64_t(sizeof(long long));
    return s;
}

template <bool HALF, class S>
static std::function<cudaError_t(cudaStream_t)> bind_moe(const MoeFusedParams& p, const CUtensorMap& in,
                                                         const CUtensorMap& out) {
    return [=](cudaStream_t stream) -> cudaError_t {
        static std::atomic<uint64_t> configured{0};  // devices whose attribute is set
        auto kern = moe_fused_kernel<HALF, S>;
        constexpr size_t smem = moe_smem_bytes<S>();
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        const uint64_t bit = uint64_t(1) << (dev & 63);
        if (!(configured.load() & bit)) {
            e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
            if (e != cudaSuccess) return e;
            configured.fetch_or(bit);
        }
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(static_cast<unsigned>(p.L.num_sms));
        cfg.blockDim = dim3(S::THREADS);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeCooperative;  // every CTA resident at once: the grid barriers can complete
        attr[0].val.cooperative = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        return cudaLaunchKernelEx(&cfg, kern, in, out, p);
    };
}

template <bool HALF, bool ALIGNED>
static std::function<cudaError_t(cudaStream_t)> bind_moe_shape(int which, const MoeFusedParams& p, const CUtensorMap& in,
                                                               const CUtensorMap& out) {
    using moe::Shape;
    switch (which) {
        case 0: return bind_moe<HALF, Shape<1, 1, ALIGNED>>(p, in, out);
        case 1: return bind_moe<HALF, Shape<1, 2, ALIGNED>>(p, in, out);
        case 2: return bind_moe<HALF, Shape<2, 2, ALIGNED>>(p, in, out);
        default: return bind_moe<HALF, Shape<4, 2, ALIGNED>>(p, in, out);
    }
}

std::function<cudaError_t(cudaStream_t)> prepare_moe_fused(const MoeLaunch& L, cudaError_t* err) {
    MoeFusedParams p = {};
    p.L = L;
    p.chunks_in = chunks_of(L.model);
    p.chunks_out = chunks_of(L.expert);
    const MoeChoice shape = moe_choice(L);
    const int rows_in = (L.gated ? 8 : 16) * shape.mt, rows_out = 16 * shape.mt;
    p.blocks_in = (L.expert + rows_in - 1) / rows_in;
    p.blocks_out = (L.model + rows_out - 1) / rows_out;
    const int64_t router_units = int64_t(L.experts) * ((L.tokens + 7) / 8);
    p.router_split = 1;
    while (p.router_split < shape.warps && router_units * p.router_split * 2 <= int64_t(L.num_sms) * shape.warps)
        p.router_split *= 2;
    auto four = [](const void* q, int half) { return (reinterpret_cast<uintptr_t>(q) & (half ? 7 : 15)) == 0; };
    p.vec = four(L.x, L.x_half) && four(L.router, L.router_half) && L.model % 4 == 0;
    p.hidden_pitch = round4(L.expert);
    p.out_pitch = round4(L.model);
    p.end_in = L.w_in + int64_t(L.experts) * (L.gated ? 2 : 1) * L.expert * L.model;
    p.end_out = L.w_out + int64_t(L.experts) * L.model * L.expert;
    const uint64_t d = L.model, f = L.expert, e = L.experts;
    CUtensorMap in = {}, out = {};
    const bool aligned = moe_aligned(L);
    const bool ok = !aligned ||
                    (make_tensor_map_u8(&in, L.w_in, d, f, (L.gated ? 2 : 1) * e, d, d * f, moe::CHUNK, rows_in,
                                       L.gated ? 2 : 1) &&
                    make_tensor_map_u8(&out, L.w_out, f, d, e, f, d * f, moe::CHUNK, rows_out));
    *err = ok ? cudaSuccess : cudaErrorInvalidValue;
    if (!ok) return nullptr;
    const int which = shape.mt == 1 ? 0 : shape.nt;
    if (aligned) return L.x_half ? bind_moe_shape<true, true>(which, p, in, out) : bind_moe_shape<false, true>(which, p, in, out);
    return L.x_half ? bind_moe_shape<true, false>(which, p, in, out) : bind_moe_shape<false, false>(which, p, in, out);
}

}  // namespace og
