// Copies of operands whose rows do not start on 16-byte boundaries into pitched buffers whose rows do, both operands of a
// product in one launch.
//
// Bound by memory traffic and, for the sizes of a decode step, by the launch itself: a thread loads the two aligned
// 16-byte units around each 16 bytes of a row, shifts them together and stores one aligned unit (a source unit is read by
// two neighbouring lanes, the second time from L1). The copy engine's two-dimensional copies, which these replace, take
// 8 us and more each and far longer for many short rows.
#include <cuda_runtime.h>

#include <algorithm>

#include "og_gemm.h"
#include "og_ptx.cuh"

namespace og {

namespace stage {
constexpr int THREADS = 256;
constexpr int UNITS = 4;  // 16-byte units per thread and pass, all loads in flight
}  // namespace stage

// Units lo, hi (hi continues lo) from byte `skew` (0 .. 15) of lo on.
__device__ __forceinline__ uint4 joined(const uint4& lo, const uint4& hi, uint32_t skew) {
    uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    if (skew & 8) {
#pragma unroll
        for (int i = 0; i < 6; i++) w[i] = w[i + 2];
    }
    if (skew & 4) {
#pragma unroll
        for (int i = 0; i < 5; i++) w[i] = w[i + 1];
    }
    const uint32_t bits = (skew & 3) * 8;
    return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                      __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
}

__global__ void __launch_bounds__(stage::THREADS) stage_kernel(const StageJob a, const StageJob b) {
    pdl_trigger();
    pdl_wait();
    const bool second = blockIdx.x >= static_cast<unsigned>(a.blocks);
    const StageJob& j = second ? b : a;
    const int64_t block = blockIdx.x - (second ? a.blocks : 0);
    const int tx = threadIdx.x & ((1 << j.lanes_log2) - 1), ty = threadIdx.x >> j.lanes_log2;
    const int64_t row = block * (stage::THREADS >> j.lanes_log2) + ty;
    if (row >= j.rows * j.batches) return;
    const int64_t batch = j.batches == 1 ? 0 : row / j.rows;
    const uintptr_t from = reinterpret_cast<uintptr_t>(j.src) + batch * j.stride + (row - batch * j.rows) * j.ld;
    const uintptr_t end = from + j.width;  // units that start past the row are not touched
    uint4* to = reinterpret_cast<uint4*>(j.dst + row * j.pitch);
    const uint32_t skew = from & 15;
    const int units = static_cast<int>(j.pitch >> 4), step = 1 << j.lanes_log2;
    for (int u0 = tx; u0 < units; u0 += stage::UNITS * step) {
        uint4 lo[stage::UNITS], hi[stage::UNITS];
#pragma unroll
        for (int i = 0; i < stage::UNITS; i++) {
            const int u = u0 + i * step;
            const uintptr_t at = (from - skew) + 16 * static_cast<uintptr_t>(u);
            lo[i] = hi[i] = make_uint4(0, 0, 0, 0);
            if (u < units) {
                lo[i] = __ldg(reinterpret_cast<const uint4*>(at));
                if (skew != 0 && at + 16 < end) hi[i] = __ldg(reinterpret_cast<const uint4*>(at + 16));
            }
        }
#pragma unroll
        for (int i = 0; i < stage::UNITS; i++)
            if (u0 + i * step < units) to[u0 + i * step] = joined(lo[i], hi[i], skew);
    }
}

cudaError_t launch_stage(StageJob a, StageJob b, cudaStream_t stream) {
    for (StageJob* j : {&a, &b}) {
        if (j->src == nullptr) continue;  // zero blocks
        const int64_t units = j->pitch >> 4;
        while (j->lanes_log2 < 8 && (int64_t(stage::UNITS) << j->lanes_log2) < units) j->lanes_log2++;
        const int64_t rows = stage::THREADS >> j->lanes_log2;
        j->blocks = (j->rows * j->batches + rows - 1) / rows;
    }
    if (a.blocks + b.blocks > 0x7FFFFFFF) return cudaErrorInvalidValue;
    return launch_pdl(stage_kernel, dim3(static_cast<unsigned>(a.blocks + b.blocks)), dim3(stage::THREADS), 0, stream, a, b);
}

}  // namespace og
