// The mixture-of-experts layer as one cooperative kernel (a CTA of 16 warps per SM), for weights TMA can load.
//
// For a few tokens the layer is bound by reading the touched experts' weights once (3 x model x expert bytes each when
// gated), so everything is arranged around keeping those reads in flight:
//  0. Router: logits (a CTA per expert and 8 tokens, its warps splitting the sum), and x rewritten as 16-bit pieces in
//     the order the matrix instructions take them. Grid barrier.
//     Every CTA then finds all tokens' experts itself (a warp per token) and sorts the (token, choice) pairs by expert
//     into groups of one expert and up to 8 NT pairs: cheaper than another barrier.
//  1. Input products: units of one group and 16 rows of w_in (8 of each half when gated, so that a lane holds both
//     factors of a hidden value), K in chunks of 128 bytes. Hidden values leave as pieces. Grid barrier.
//  2. Output products: units of one group and 16 rows of w_out; weighted results per pair. Grid barrier.
//  3. The sum over each token's pairs, in the order of their rank: the result does not depend on the schedule.
// A CTA owns a contiguous range of units and its warps equal contiguous ranges of the units' chunks; a unit cut between
// warps meets through partial sums (`segments`), added in order by the warp that holds its start. Each warp
// feeds itself: a ring of SLOTS 2 KB boxes loaded by TMA (128-byte swizzle, no multicast), the next box issued as soon as
// one is in registers. The ring runs on into phase 2's weights, which do not depend on the barrier: DRAM stays busy
// while the hidden values are exchanged.
//
// Arithmetic: int8 weights are exact in 16 bits. float16 x multiplies as it is; float32 values are cut into three
// bfloat16 pieces of 8 bits (exact), hidden values of a float16 layer into two (16 bits, 2^-17 relative, the range of
// float32). mma.sync m16n8k16 with the weights as the 16-row operand and 8 tokens as its columns: the tensor
// cores' rate does not matter here (one token per expert uses an eighth of a tile), the fragments come straight from
// the swizzled rows, and 128-row tcgen05 tiles would cut the work too coarsely for one token. Every chunk's sums start
// at zero and are added in float32, so that no more than 128 products are accumulated inside the matrix instructions.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "og_act.cuh"
#include "og_gemm.h"
#include "og_moe.h"
#include "og_ptx.cuh"

namespace og {

namespace moe {
constexpr int WARPS = 16;
constexpr int THREADS = 32 * WARPS;
constexpr int ROWS = 16;                      // weight rows of a unit
constexpr int CHUNK = 128;                    // bytes of K of a box
constexpr int BOX = ROWS * CHUNK;             // 2 KB
constexpr int SLOTS = 4;                      // boxes in flight per warp: 128 KB per SM
constexpr int MAX_PAIRS = MOE_MAX_TOKENS * MOE_MAX_TOP_K;
constexpr int PIECE_BYTES = 2 * CHUNK;        // one piece of one row's chunk
}  // namespace moe

struct MoeFusedParams {
    MoeLaunch L;
    int chunks_in, chunks_out;  // K chunks of the two products
    int blocks_in, blocks_out;  // units per group
};

// A group: one expert and a run of the pairs sorted by expert.
struct MoeGroup {
    uint16_t expert, first, count, pad;
};

template <int NT>
struct MoeShared {
    static constexpr int GROUPS = MOE_MAX_EXPERTS + moe::MAX_PAIRS / (8 * NT);
    uint64_t full[moe::WARPS][moe::SLOTS];
    double logit_part[2][moe::WARPS][8];
    float weight[moe::MAX_PAIRS];      // by pair (token * top_k + rank)
    uint16_t id[moe::MAX_PAIRS];       // by pair
    uint16_t order[moe::MAX_PAIRS];    // pairs sorted by expert
    MoeGroup group[GROUPS];
    int warp_total[2][moe::WARPS];
    int groups;
    int abort;
    int failed;
};

template <int NT>
__host__ __device__ constexpr int moe_segment_floats() { return moe::ROWS * 8 * NT; }

template <int NT>
constexpr size_t moe_smem_bytes() {
    return 1024 + size_t(moe::WARPS) * moe::SLOTS * moe::BOX + sizeof(MoeShared<NT>);
}

// ---- pieces ---------------------------------------------------------------------------------------------------------

// A float32 as P 16-bit pieces whose sum it is: for P = 1 the float16 it came from; for P = 3 three bfloat16 of 8 bits,
// cut off rather than rounded so that no piece overflows; for P = 2 the second one rounded. An infinity or NaN is its
// first piece alone.
template <int P>
__device__ __forceinline__ void to_pieces(float v, uint16_t (&out)[P]) {
    if constexpr (P == 1) {
        out[0] = __half_as_ushort(__float2half_rn(v));
    } else {
        const uint32_t bits = __float_as_uint(v);
        if ((bits & 0x7F800000u) == 0x7F800000u) {
            out[0] = static_cast<uint16_t>((bits & 0x007FFFFFu) ? 0x7FC0u : bits >> 16);
#pragma unroll
            for (int p = 1; p < P; p++) out[p] = 0;
            return;
        }
#pragma unroll
        for (int p = 0; p < P; p++) {
            if (P == 2 && p == 1) {
                out[p] = __bfloat16_as_ushort(__float2bfloat16_rn(v));
            } else {
                const uint32_t top = __float_as_uint(v) & 0xFFFF0000u;
                out[p] = static_cast<uint16_t>(top >> 16);
                v = v - __uint_as_float(top);  // exact
            }
        }
    }
}

// Two bytes of a word of int8 weights as a pair of 16-bit floats, exactly. float16: 0x6400 | u is 1024 + u for the byte
// u = w + 128. bfloat16 holds 7 mantissa bits: 0x4300 | (w & 0x7F) is 128 + those bits, and 0x4300 | (w & 0x80) is 128, or
// 256 for a negative w.
template <bool BF16, bool HIGH>
__device__ __forceinline__ uint32_t weight_pair(uint32_t w) {
    uint32_t r;
    if constexpr (BF16) {
        const uint32_t p = __byte_perm(w, 0x43434343u, HIGH ? 0x4342 : 0x4140);
        const uint32_t a = p & 0xFF7FFF7Fu, b = p & 0xFF80FF80u;
        const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                         *reinterpret_cast<const __nv_bfloat162*>(&b));
        r = *reinterpret_cast<const uint32_t*>(&d);
    } else {
        const uint32_t p = __byte_perm(w, 0x64646464u, HIGH ? 0x4342 : 0x4140);  // w: bytes + 128
        const uint32_t b = 0x64806480u;                                          // 1152
        const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&p), *reinterpret_cast<const __half2*>(&b));
        r = *reinterpret_cast<const uint32_t*>(&d);
    }
    return r;
}

template <bool BF16>
__device__ __forceinline__ void moe_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ---- grid barrier ---------------------------------------------------------------------------------------------------

// Every CTA of the launch arrives; `wait` false only arrives (a CTA that has failed keeps the count whole for the
// others and for later launches). Bounded; false when it gave up.
__device__ __forceinline__ bool grid_arrive(unsigned long long* arrivals, bool wait) {
    __threadfence();
    const unsigned G = gridDim.x;
    const unsigned long long before = atomicAdd(arrivals, 1ull);
    if (!wait) return true;
    const unsigned long long target = (before / G + 1ull) * G;
    if (before + 1ull != target) {
        const uint64_t t0 = global_timer_ns();
        while (true) {
            unsigned long long now;
            asm volatile("ld.acquire.gpu.global.u64 %0, [%1];" : "=l"(now) : "l"(arrivals) : "memory");
            if (now >= target) break;
            if (global_timer_ns() - t0 > OG_WAIT_LIMIT_NS) return false;
        }
    }
    __threadfence();
    return true;
}

// The whole CTA meets the grid; false (for every thread) when this CTA has failed or gives up here.
template <class S>
__device__ __forceinline__ bool grid_barrier(S& sh, unsigned long long* arrivals) {
    __syncthreads();
    if (threadIdx.x == 0) {
        const bool ok = sh.abort == 0;
        if (!grid_arrive(arrivals, ok) || !ok) sh.failed = 1;
    }
    __syncthreads();
    return sh.failed == 0;
}

// ---- phase 0 --------------------------------------------------------------------------------------------------------

__device__ __forceinline__ float moe_load(const void* p, int half, int64_t i) {
    return half ? __half2float(__ldg(static_cast<const __half*>(p) + i)) : __ldg(static_cast<const float*>(p) + i);
}

// x as pieces: 16-byte unit (j, q) of a chunk's piece holds the eight values k = 32 q + 8 j ..; and zeros in the part of
// the hidden values' last chunk that lies past the expert's size.
template <int PX, int PH>
__device__ __forceinline__ void moe_split_x(const MoeFusedParams& p) {
    const MoeLaunch& L = p.L;
    const int thread = blockIdx.x * moe::THREADS + threadIdx.x, threads = gridDim.x * moe::THREADS;
    const int units = L.tokens * p.chunks_in * 16;
    for (int u = thread; u < units; u += threads) {
        const int t = u / (p.chunks_in * 16), c = (u >> 4) % p.chunks_in, j = (u >> 2) & 3, q = u & 3;
        const int k0 = c * moe::CHUNK + 32 * q + 8 * j;
        uint16_t piece[PX][8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            uint16_t v[PX];
            to_pieces<PX>(k0 + i < L.model ? moe_load(L.x, L.x_half, static_cast<int64_t>(t) * L.model + k0 + i) : 0.0f, v);
#pragma unroll
            for (int s = 0; s < PX; s++) piece[s][i] = v[s];
        }
        uint8_t* to = L.x_pieces + (static_cast<int64_t>(t) * p.chunks_in + c) * PX * moe::PIECE_BYTES + j * 64 + q * 16;
#pragma unroll
        for (int s = 0; s < PX; s++)
            *reinterpret_cast<uint4*>(to + s * moe::PIECE_BYTES) =
                make_uint4(piece[s][0] | piece[s][1] << 16, piece[s][2] | piece[s][3] << 16,
                           piece[s][4] | piece[s][5] << 16, piece[s][6] | piece[s][7] << 16);
    }
    const int used = (L.expert % moe::CHUNK) / 8;  // units of the last chunk that hold values (expert is a multiple of 8)
    if (used != 0) {
        const int pairs = L.tokens * L.top_k, empty = 16 - used;
        for (int u = thread; u < pairs * empty * PH; u += threads) {
            const int pair = u / (empty * PH), s = (u / empty) % PH, k = 8 * (used + u % empty);
            uint8_t* to = L.h_pieces +
                          ((static_cast<int64_t>(pair) * p.chunks_out + p.chunks_out - 1) * PH + s) * moe::PIECE_BYTES +
                          (k % 32) / 8 * 64 + k / 32 * 16;
            *reinterpret_cast<uint4*>(to) = make_uint4(0, 0, 0, 0);
        }
    }
}

// Logits: a CTA per (expert, 8 tokens), lanes striding over the sum; eight products at a time in float32, the rest in
// float64, so that near-equal logits rank as their exact values do.
template <class S>
__device__ __forceinline__ void moe_logits(const MoeLaunch& L, S& sh) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int token_blocks = (L.tokens + 7) / 8;
    int buffer = 0;
    for (int unit = blockIdx.x; unit < L.experts * token_blocks; unit += gridDim.x, buffer ^= 1) {
        const int e = unit / token_blocks, t0 = (unit % token_blocks) * 8, n = min(8, L.tokens - t0);
        double sum[8];
#pragma unroll
        for (int i = 0; i < 8; i++) sum[i] = 0.0;
        for (int d0 = threadIdx.x; d0 < L.model; d0 += 8 * moe::THREADS) {
            float part[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < 8; s++) {
                const int d = d0 + s * moe::THREADS;
                if (d >= L.model) break;
                const float r = moe_load(L.router, L.router_half, static_cast<int64_t>(e) * L.model + d);
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (i < n) part[i] = fmaf(moe_load(L.x, L.x_half, static_cast<int64_t>(t0 + i) * L.model + d), r, part[i]);
            }
#pragma unroll
            for (int i = 0; i < 8; i++) sum[i] += part[i];
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
        if (static_cast<int>(threadIdx.x) < n) {
            double total = 0.0;
            for (int w = 0; w < moe::WARPS; w++) total += sh.logit_part[buffer][w][threadIdx.x];
            L.logits[static_cast<int64_t>(t0 + threadIdx.x) * L.experts + e] = static_cast<float>(total);
        }
    }
}

// ---- routing --------------------------------------------------------------------------------------------------------

// A key that orders floats as unsigned numbers; NaN below every number, with -infinity (what it ranks as).
__device__ __forceinline__ uint32_t rank_key(float v) {
    const uint32_t u = __float_as_uint(isnan(v) ? -INFINITY : (v == 0.0f ? 0.0f : v));
    return u & 0x80000000u ? ~u : u | 0x80000000u;  // -infinity is 0x007FFFFF: 0 marks a taken expert
}

// A token's experts by one warp: the largest key, the lowest expert among equals, top_k times.
template <class S>
__device__ __forceinline__ void moe_choose(const MoeLaunch& L, S& sh, int t, bool publish) {
    const int lane = threadIdx.x & 31;
    constexpr int PER_LANE = MOE_MAX_EXPERTS / 32;
    const float* logits = L.logits + static_cast<int64_t>(t) * L.experts;
    uint32_t key[PER_LANE];
    float top = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < PER_LANE; i++) {
        key[i] = 0;
        if (32 * i < L.experts && lane + 32 * i < L.experts) {
            const float v = __ldcg(logits + lane + 32 * i);
            key[i] = rank_key(v);
            nan |= isnan(v);
            top = fmaxf(top, v);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    if (__any_sync(0xFFFFFFFFu, nan)) top = NAN;  // the softmax of a row with a NaN is NaN
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < PER_LANE; i++)
        if (32 * i < L.experts && lane + 32 * i < L.experts) sum += expf(__ldcg(logits + lane + 32 * i) - top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    float weight = 0.0f, chosen = 0.0f;
    int id = 0;
    for (int k = 0; k < L.top_k; k++) {
        uint32_t best = 0;
#pragma unroll
        for (int i = 0; i < PER_LANE; i++)
            if (32 * i < L.experts) best = max(best, key[i]);
        best = __reduce_max_sync(0xFFFFFFFFu, best);
        int at = MOE_MAX_EXPERTS;
#pragma unroll
        for (int i = PER_LANE - 1; i >= 0; i--)
            if (32 * i < L.experts && key[i] == best) at = lane + 32 * i;
        at = __reduce_min_sync(0xFFFFFFFFu, at);
#pragma unroll
        for (int i = 0; i < PER_LANE; i++)
            if (at == lane + 32 * i) key[i] = 0;
        const float w = expf(__ldcg(logits + at) - top) / sum;
        chosen += w;
        if (lane == k) {
            weight = w;
            id = at;
        }
    }
    if (lane < L.top_k) {
        if (L.normalize) weight = weight / chosen;
        const int i = t * L.top_k + lane;
        sh.id[i] = static_cast<uint16_t>(id);
        sh.weight[i] = weight;
        if (publish) {
            if (L.ids_out != nullptr) L.ids_out[i] = id;
            if (L.weights_out != nullptr) L.weights_out[i] = weight;
        }
    }
}

// The pairs sorted by expert and cut into groups of at most 8 NT pairs: thread e counts, places and lists expert e.
template <int NT>
__device__ __forceinline__ void moe_group(const MoeLaunch& L, MoeShared<NT>& sh) {
    const int e = threadIdx.x, warp = e >> 5, lane = e & 31;
    const int pairs = L.tokens * L.top_k;
    int count = 0;
    if (e < L.experts)
        for (int i = 0; i < pairs; i++) count += sh.id[i] == e;
    const int groups = (count + 8 * NT - 1) / (8 * NT);
    int first = count, group = groups;  // inclusive sums over the experts
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
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
    for (int w = 0; w < warp; w++) {
        first += sh.warp_total[0][w];
        group += sh.warp_total[1][w];
    }
    if (e == moe::THREADS - 1) sh.groups = group;
    first -= count;
    group -= groups;
    if (count > 0) {
        int at = first;
        for (int i = 0; i < pairs; i++)
            if (sh.id[i] == e) sh.order[at++] = static_cast<uint16_t>(i);
        for (int g = 0; g < groups; g++)
            sh.group[group + g] = MoeGroup{static_cast<uint16_t>(e), static_cast<uint16_t>(first + g * 8 * NT),
                                           static_cast<uint16_t>(min(8 * NT, count - g * 8 * NT)), 0};
    }
    __syncthreads();
}

// ---- phases 1 and 2 -------------------------------------------------------------------------------------------------

// One phase's work of this warp: chunks [at, end) of the CTA's units, unit u0 + i / chunks, chunk i % chunks.
struct MoeRange {
    int u0, units;  // the CTA's units
    int at, end;
};

__device__ __forceinline__ int moe_split(int total, int part, int parts) {
    return static_cast<int>(static_cast<int64_t>(total) * part / parts);
}

__device__ __forceinline__ MoeRange moe_range(int units, int chunks, int warp) {
    MoeRange r;
    r.u0 = moe_split(units, blockIdx.x, gridDim.x);
    r.units = moe_split(units, blockIdx.x + 1, gridDim.x) - r.u0;
    r.at = moe_split(r.units * chunks, warp, moe::WARPS);
    r.end = moe_split(r.units * chunks, warp + 1, moe::WARPS);
    return r;
}

// The warp that holds chunk i of `total`.
__device__ __forceinline__ int moe_owner(int i, int total) {
    return static_cast<int>((static_cast<int64_t>(i + 1) * moe::WARPS - 1) / total);
}

// What the warp's ring loads next: phase 1's range, then phase 2's.
struct MoeFeed {
    int phase, at, end;
    uint32_t issued;  // boxes so far
};

template <int NT>
struct MoeWarp {
    const MoeFusedParams& p;
    MoeShared<NT>& sh;
    const CUtensorMap* maps[2];
    uint8_t* ring;
    uint64_t* full;
    int lane;
    MoeRange range[2];
    MoeFeed feed;
    uint32_t taken;  // boxes read so far

    __device__ __forceinline__ int chunks(int phase) const { return phase == 0 ? p.chunks_in : p.chunks_out; }
    __device__ __forceinline__ int blocks(int phase) const { return phase == 0 ? p.blocks_in : p.blocks_out; }

    // Issues the next box, if any is left and a slot is free.
    __device__ __forceinline__ void issue() {
        while (feed.phase < 2 && feed.at >= feed.end) {
            feed.phase++;
            if (feed.phase < 2) {
                feed.at = range[1].at;
                feed.end = range[1].end;
            }
        }
        if (feed.phase >= 2 || feed.issued - taken >= moe::SLOTS) return;
        const int c = chunks(feed.phase), b = blocks(feed.phase);
        const int local = feed.at / c, chunk = feed.at - local * c;
        const int unit = range[feed.phase].u0 + local, g = unit / b, block = unit - g * b;
        if (lane == 0) {
            const int slot = feed.issued % moe::SLOTS;
            const int e = sh.group[g].expert;
            const bool halves = feed.phase == 0 && p.L.gated;
            mbar_arrive_expect_tx(&full[slot], moe::BOX);
            tma_load_3d(ring + slot * moe::BOX, maps[feed.phase], &full[slot], chunk * moe::CHUNK,
                        block * (halves ? 8 : 16), halves ? 2 * e : e);
        }
        feed.at++;
        feed.issued++;
    }

    // The sums of one unit's chunks [c0, c1) for the group's columns: row g (and g + 8) of the unit, columns 2 q and
    // 2 q + 1 of n-tile t in acc[t]. BF16 and P: the pieces of the columns' values at `values`, `row` by column.
    template <bool BF16, int P>
    __device__ __forceinline__ bool products(const uint8_t* values, const uint32_t (&row)[NT], int tiles, int c0, int c1,
                                             float (&acc)[NT][4]) {
        const int g = lane >> 2, q = lane & 3;
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[t][i] = 0.0f;
#pragma unroll 1
        for (int c = c0; c < c1; c++) {
            const int slot = taken % moe::SLOTS;
            const bool ok = mbar_wait(&full[slot], (taken / moe::SLOTS) & 1, &sh.abort);
            if (!__all_sync(0xFFFFFFFFu, ok)) return false;
            // Bytes 32 q .. 32 q + 31 of rows g and g + 8: 16-byte units 2 q and 2 q + 1, swizzled by the row. Eight
            // consecutive lanes touch eight different units of 128 bytes: no bank conflict.
            const uint8_t* box = ring + slot * moe::BOX + g * moe::CHUNK;
            uint4 w[2][2];
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int u = 0; u < 2; u++)
                    w[h][u] = *reinterpret_cast<const uint4*>(box + h * 8 * moe::CHUNK + (((2 * q + u) ^ g) << 4));
            taken++;
            __syncwarp();  // the slot is in registers
            issue();
            uint32_t a[8][4];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const uint32_t lo[4] = {w[0][u].x, w[0][u].y, w[0][u].z, w[0][u].w};
                const uint32_t hi[4] = {w[1][u].x, w[1][u].y, w[1][u].z, w[1][u].w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t x = BF16 ? lo[i] : lo[i] ^ 0x80808080u, y = BF16 ? hi[i] : hi[i] ^ 0x80808080u;
                    a[4 * u + i][0] = weight_pair<BF16, false>(x);
                    a[4 * u + i][1] = weight_pair<BF16, false>(y);
                    a[4 * u + i][2] = weight_pair<BF16, true>(x);
                    a[4 * u + i][3] = weight_pair<BF16, true>(y);
                }
            }
#pragma unroll
            for (int t = 0; t < NT; t++) {
                if (t >= tiles) break;
                const uint8_t* v = values + row[t] + c * P * moe::PIECE_BYTES + q * 16;
                float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int piece = P - 1; piece >= 0; piece--) {  // the smallest first
                    uint4 b[4];
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        b[j] = *reinterpret_cast<const uint4*>(v + piece * moe::PIECE_BYTES + j * 64);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        moe_mma<BF16>(s, a[2 * j], b[j].x, b[j].y);
                        moe_mma<BF16>(s, a[2 * j + 1], b[j].z, b[j].w);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; i++) acc[t][i] += s[i];
            }
        }
        return true;
    }

    // Phase 1's results: rows g and g + 8 of the unit times their scales; the hidden values as pieces.
    template <int PH>
    __device__ __forceinline__ void finish_in(int unit, const float (&acc)[NT][4]) {
        const MoeLaunch& L = p.L;
        const int g = lane >> 2, q = lane & 3;
        const MoeGroup grp = sh.group[unit / p.blocks_in];
        const int block = unit % p.blocks_in;
        const int j0 = L.gated ? block * 8 + g : block * 16 + g;
        const int64_t rows = static_cast<int64_t>(L.gated ? 2 : 1) * L.expert;
        const float* scale = L.in_scale + grp.expert * rows;
        const float s0 = j0 < L.expert ? __ldg(scale + j0) : 0.0f;
        const int j1 = L.gated ? j0 + L.expert : j0 + 8;
        const float s1 = (L.gated ? j0 < L.expert : j1 < L.expert) ? __ldg(scale + j1) : 0.0f;
#pragma unroll
        for (int t = 0; t < NT; t++) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int n = 8 * t + 2 * q + i;
                if (n >= grp.count) continue;
                const int pair = sh.order[grp.first + n];
                float h[2] = {acc[t][i] * s0, acc[t][2 + i] * s1};
                if (L.gated) {
                    float f[1] = {h[0]};
                    activate_all(f, L.activation);
                    if (j0 < L.expert) put_hidden<PH>(pair, j0, f[0] * h[1]);
                } else {
                    activate_all(h, L.activation);
                    if (j0 < L.expert) put_hidden<PH>(pair, j0, h[0]);
                    if (j1 < L.expert) put_hidden<PH>(pair, j1, h[1]);
                }
            }
        }
    }

    template <int PH>
    __device__ __forceinline__ void put_hidden(int pair, int j, float v) {
        uint16_t piece[PH];
        to_pieces<PH>(v, piece);
        const int k = j % moe::CHUNK;
        uint8_t* to = p.L.h_pieces + (static_cast<int64_t>(pair) * p.chunks_out + j / moe::CHUNK) * PH * moe::PIECE_BYTES +
                      (k % 32) / 8 * 64 + k / 32 * 16 + (k % 8) * 2;
#pragma unroll
        for (int s = 0; s < PH; s++) *reinterpret_cast<uint16_t*>(to + s * moe::PIECE_BYTES) = piece[s];
    }

    // Phase 2's results: the pair's weight times the row's scale times the sum.
    __device__ __forceinline__ void finish_out(int unit, const float (&acc)[NT][4]) {
        const MoeLaunch& L = p.L;
        const int g = lane >> 2, q = lane & 3;
        const MoeGroup grp = sh.group[unit / p.blocks_out];
        const int d0 = (unit % p.blocks_out) * 16 + g;
        const float* scale = L.out_scale + static_cast<int64_t>(grp.expert) * L.model;
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const int d = d0 + 8 * r;
            if (d >= L.model) continue;
            const float s = __ldg(scale + d);
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int n = 8 * t + 2 * q + i;
                    if (n >= grp.count) continue;
                    const int pair = sh.order[grp.first + n];
                    L.outputs[static_cast<int64_t>(pair) * L.model + d] = sh.weight[pair] * (acc[t][2 * r + i] * s);
                }
        }
    }

    __device__ __forceinline__ float* segment(int warp, int which) const {
        return p.L.segments + (static_cast<int64_t>(blockIdx.x * moe::WARPS + warp) * 2 + which) * moe_segment_floats<NT>();
    }

    // The warp's range of one phase. False when a wait gave up.
    template <int PHASE, bool BF16, int P, int PH>
    __device__ __forceinline__ bool run(int warp) {
        const MoeRange r = range[PHASE];
        const int c = chunks(PHASE), total = r.units * c;
        const uint8_t* values = PHASE == 0 ? p.L.x_pieces : p.L.h_pieces;
        const uint32_t row_bytes = static_cast<uint32_t>(c) * P * moe::PIECE_BYTES;
        const int g = lane >> 2;
        for (int at = r.at; at < r.end;) {
            const int local = at / c, c0 = at - local * c, c1 = min(c, c0 + r.end - at);
            const int unit = r.u0 + local;
            const MoeGroup grp = sh.group[unit / blocks(PHASE)];
            const int tiles = (grp.count + 7) / 8;
            uint32_t row[NT];
#pragma unroll
            for (int t = 0; t < NT; t++) {  // columns past the group's pairs repeat its last one and are not stored
                const int pair = sh.order[grp.first + min(8 * t + g, grp.count - 1)];
                row[t] = static_cast<uint32_t>(PHASE == 0 ? pair / p.L.top_k : pair) * row_bytes;
            }
            float acc[NT][4];
            if (!products<BF16, P>(values, row, tiles, c0, c1, acc)) break;  // the abort flag is up
            if (c0 == 0 && c1 == c) {
                if constexpr (PHASE == 0)
                    finish_in<PH>(unit, acc);
                else
                    finish_out(unit, acc);
            } else {
                float4* to = reinterpret_cast<float4*>(segment(warp, at == r.at ? 0 : 1)) + lane;
#pragma unroll
                for (int t = 0; t < NT; t++)
                    if (t < tiles) to[32 * t] = make_float4(acc[t][0], acc[t][1], acc[t][2], acc[t][3]);
            }
            at += c1 - c0;
        }
        __syncthreads();
        if (sh.abort) return false;
        // A cut unit is finished by the warp that holds its start: its own segment is its last one (or, starting at its
        // range's start, its first), the others' are their first.
        if (r.at < r.end) {
            const int local = (r.end - 1) / c, i0 = local * c;
            if (i0 >= r.at && i0 + c > r.end) {
                const int unit = r.u0 + local;
                const int tiles = (sh.group[unit / blocks(PHASE)].count + 7) / 8;
                const int last = moe_owner(i0 + c - 1, total);
                float acc[NT][4];
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) acc[t][i] = 0.0f;
                for (int w = warp; w <= last; w++) {
                    if (moe_split(total, w, moe::WARPS) == moe_split(total, w + 1, moe::WARPS)) continue;  // no share
                    const float4* from = reinterpret_cast<const float4*>(segment(w, w == warp && i0 != r.at ? 1 : 0)) + lane;
#pragma unroll
                    for (int t = 0; t < NT; t++)
                        if (t < tiles) {
                            const float4 v = from[32 * t];
                            acc[t][0] += v.x;
                            acc[t][1] += v.y;
                            acc[t][2] += v.z;
                            acc[t][3] += v.w;
                        }
                }
                if constexpr (PHASE == 0)
                    finish_in<PH>(unit, acc);
                else
                    finish_out(unit, acc);
            }
        }
        return true;
    }

    // Waits (bounded) for boxes still in flight: none may land after the CTA has gone.
    __device__ __forceinline__ void drain() {
        int give_up = 0;
        while (taken != feed.issued) {
            if (!mbar_wait(&full[taken % moe::SLOTS], (taken / moe::SLOTS) & 1, &give_up)) break;
            taken++;
        }
    }
};

template <bool HALF, int NT>
__global__ void __launch_bounds__(moe::THREADS, 1)
    moe_fused_kernel(const __grid_constant__ CUtensorMap map_in, const __grid_constant__ CUtensorMap map_out,
                     const __grid_constant__ MoeFusedParams p) {
    constexpr int PX = HALF ? 1 : 3, PH = HALF ? 2 : 3;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    MoeShared<NT>& sh = *reinterpret_cast<MoeShared<NT>*>(smem + moe::WARPS * moe::SLOTS * moe::BOX);
    const MoeLaunch& L = p.L;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_trigger();
    if (threadIdx.x == 0) {
        for (int w = 0; w < moe::WARPS; w++)
            for (int s = 0; s < moe::SLOTS; s++) mbar_init(&sh.full[w][s], 1);
        sh.abort = 0;
        sh.failed = 0;
        fence_mbar_init();
        prefetch_tmap(&map_in);
        prefetch_tmap(&map_out);
    }
    pdl_wait();
    moe_split_x<PX, PH>(p);
    moe_logits(L, sh);
    if (!grid_barrier(sh, L.arrivals)) {
        if (threadIdx.x == 0) {
            grid_arrive(L.arrivals, false);
            grid_arrive(L.arrivals, false);
            atomicExch(L.error_flag, 1);
        }
        return;
    }
    for (int t = warp; t < L.tokens; t += moe::WARPS) moe_choose(L, sh, t, blockIdx.x == 0);
    __syncthreads();
    moe_group<NT>(L, sh);

    MoeWarp<NT> me{p, sh, {&map_in, &map_out}, smem + warp * moe::SLOTS * moe::BOX, sh.full[warp], lane, {}, {}, 0};
    me.range[0] = moe_range(sh.groups * p.blocks_in, p.chunks_in, warp);
    me.range[1] = moe_range(sh.groups * p.blocks_out, p.chunks_out, warp);
    me.feed = MoeFeed{0, me.range[0].at, me.range[0].end, 0};
    for (int s = 0; s < moe::SLOTS; s++) me.issue();

    bool ok = me.template run<0, !HALF, PX, PH>(warp);
    ok = grid_barrier(sh, L.arrivals) && ok;
    if (ok) ok = me.template run<1, true, PH, PH>(warp);
    me.drain();
    if (sh.failed) {  // the same for every thread
        if (threadIdx.x == 0) {
            grid_arrive(L.arrivals, false);
            atomicExch(L.error_flag, 1);
        }
        return;
    }
    if (!grid_barrier(sh, L.arrivals)) {
        if (threadIdx.x == 0) atomicExch(L.error_flag, 1);
        return;
    }
    const int total = L.tokens * L.model / 4;  // model is a multiple of 16
    for (int i = blockIdx.x * moe::THREADS + threadIdx.x; i < total; i += gridDim.x * moe::THREADS) {
        const int t = i / (L.model / 4), d = (i - t * (L.model / 4)) * 4;
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int k = 0; k < L.top_k; k++) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(
                L.outputs + (static_cast<int64_t>(t) * L.top_k + k) * L.model + d));
            sum.x += v.x;
            sum.y += v.y;
            sum.z += v.z;
            sum.w += v.w;
        }
        const float out[4] = {sum.x, sum.y, sum.z, sum.w};
        const int64_t at = static_cast<int64_t>(t) * L.model + d;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            if constexpr (HALF) {
                const float r = L.residual != nullptr ? __half2float(static_cast<const __half*>(L.residual)[at + u]) : 0.0f;
                static_cast<__half*>(L.y)[at + u] = __float2half_rn(out[u] + r);
            } else {
                const float r = L.residual != nullptr ? static_cast<const float*>(L.residual)[at + u] : 0.0f;
                static_cast<float*>(L.y)[at + u] = out[u] + r;
            }
        }
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------

static int moe_tiles(const MoeLaunch& L) { return L.tokens <= 8 ? 1 : 4; }

static int chunks_of(int size) { return (size + moe::CHUNK - 1) / moe::CHUNK; }

bool moe_fused_eligible(const MoeLaunch& L) {
    auto aligned = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
    return L.model % 16 == 0 && L.expert % 16 == 0 && aligned(L.w_in) && aligned(L.w_out);
}

MoeFusedSizes moe_fused_sizes(const MoeLaunch& L) {
    const int64_t pairs = int64_t(L.tokens) * L.top_k;
    MoeFusedSizes s;
    s.logits = int64_t(L.tokens) * L.experts * 4;
    s.x_pieces = int64_t(L.tokens) * chunks_of(L.model) * (L.x_half ? 1 : 3) * moe::PIECE_BYTES;
    s.h_pieces = pairs * chunks_of(L.expert) * (L.x_half ? 2 : 3) * moe::PIECE_BYTES;
    s.outputs = pairs * L.model * 4;
    s.segments = int64_t(L.num_sms) * moe::WARPS * 2 * moe::ROWS * 8 * moe_tiles(L) * 4;
    return s;
}

template <bool HALF, int NT>
static std::function<cudaError_t(cudaStream_t)> bind_moe(const MoeFusedParams& p, const CUtensorMap& in,
                                                         const CUtensorMap& out) {
    return [=](cudaStream_t stream) -> cudaError_t {
        static std::atomic<uint64_t> configured{0};  // devices whose attribute is set
        auto kern = moe_fused_kernel<HALF, NT>;
        constexpr size_t smem = moe_smem_bytes<NT>();
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
        cfg.blockDim = dim3(moe::THREADS);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeCooperative;  // every CTA resident at once: the grid barriers can complete
        attr[0].val.cooperative = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        e = cudaLaunchKernelEx(&cfg, kern, in, out, p);
        if (e != cudaErrorCooperativeLaunchTooLarge) return e;
        cudaGetLastError();  // refused before anything ran
        return launch_moe_portable(p.L, stream);
    };
}

std::function<cudaError_t(cudaStream_t)> prepare_moe_fused(const MoeLaunch& L, cudaError_t* err) {
    MoeFusedParams p = {};
    p.L = L;
    p.chunks_in = chunks_of(L.model);
    p.chunks_out = chunks_of(L.expert);
    p.blocks_in = L.gated ? (L.expert + 7) / 8 : (L.expert + 15) / 16;
    p.blocks_out = (L.model + 15) / 16;
    const uint64_t d = L.model, f = L.expert, e = L.experts;
    CUtensorMap in, out;
    const bool ok = make_tensor_map_u8(&in, L.w_in, d, f, (L.gated ? 2 : 1) * e, d, d * f, moe::CHUNK, L.gated ? 8 : 16,
                                       L.gated ? 2 : 1) &&
                    make_tensor_map_u8(&out, L.w_out, f, d, e, f, d * f, moe::CHUNK, 16);
    *err = ok ? cudaSuccess : cudaErrorInvalidValue;
    if (!ok) return nullptr;
    const bool one = moe_tiles(L) == 1;
    if (L.x_half) return one ? bind_moe<true, 1>(p, in, out) : bind_moe<true, 4>(p, in, out);
    return one ? bind_moe<false, 1>(p, in, out) : bind_moe<false, 4>(p, in, out);
}

}  // namespace og
