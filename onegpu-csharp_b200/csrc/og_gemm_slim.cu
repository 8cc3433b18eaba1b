// The activated int8 product for few rows (one token to a few hundred), bound by reading B once.
//
// As in the few-rows kernel the operands' roles are swapped: the MMA computes D[n, j] = sum_k B[k, n] A[j, k] with
// tcgen05.mma.kind::i8, M = 128 columns of B and N = MR rows of A (16, 32, 64 or 128; TMA zero-fills the rows past M), and
// a second N = 16 MMA against a block of ones gives the column sums of B when A has a zero point. A cluster of P CTAs
// shares one column tile, each taking a P-th of K, so that any N occupies the SMs (two CTAs on each); the CTAs' sums
// meet in shared memory: every CTA leaves its 128 x MR partial sums in its own (the operand ring, idle by then), and
// finishes every P-th row from all of them. Against whole tiles (128 x 256 per CTA: 32 CTAs for 8192 columns) and against
// the even split with records in global memory and a ticket per tile: see the rule in slim_parts.
//
// Warp 0 loads (TMA, no multicast), warp 1 issues the MMAs, warps 2-5 sum the rows of A in the boxes (the zero
// point of B needs them), then drain TMEM (lane = column) and finish: stores and residual reads run
// along N. Every wait on an mbarrier is bounded; the cluster's own barriers are always reached, by CTAs that gave up too.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "og_gemm.h"
#include "og_kernels.cuh"
#include "og_ptx.cuh"

namespace og {

namespace slim {
constexpr int BN = 128;  // columns of B (rows of the MMA) per CTA
constexpr int BK = 128;
constexpr int MAX_PARTS = 8;
constexpr int THREADS = 192;
constexpr int FINISH_THREADS = 128;

template <int MR>
struct Cfg {
    static constexpr int B_BYTES = BN * BK;     // 16 KB
    static constexpr int A_BYTES = MR * BK;
    static constexpr int ONES_BYTES = 16 * BK;  // 16 rows of ones, shared by every stage
    static constexpr int STAGES = MR >= 128 ? 3 : 4;
    // Accumulators, taken in turn by the K = 32 steps of a block: short MMAs would wait for one another on one.
    static constexpr int ACCS = MR == 16 ? 4 : MR == 128 ? 1 : 2;
    static constexpr int ACC_COLS = MR + 16;    // dot products, then column sums of B
    static constexpr int TMEM_COLS = ACCS * ACC_COLS <= 128 ? 128 : 256;
    static constexpr int RING = STAGES * (B_BYTES + A_BYTES);
    static constexpr int SMEM_BYTES = RING + ONES_BYTES + 1024 /* alignment */ + 256 /* barriers */ + 4 * (BN + 4 * MR);
    static_assert(MR * BN * 4 <= RING, "the partial sums fit the ring");
    static_assert(2 * TMEM_COLS <= 512 && 2 * (SMEM_BYTES + 1024) <= 227 * 1024, "two CTAs on an SM");
};
}  // namespace slim

struct SlimParams {
    int m, n, k;
    int k_blocks;
    int tiles, row_chunks;  // column tiles and chunks of MR rows of one batch
    int a_batched, b_batched;
    Epilogue epi;
    int* error_flag;
    uint64_t wait_limit_ns;
    int withhold;  // watchdog self-test: the first CTA leaves its last load out
};

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr));  // after the cluster's barrier
    return v;
}

__device__ __forceinline__ int32_t byte_sum(const uint4& v, int is_signed, int32_t sum) {
    const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; j++)
        sum = is_signed ? __dp4a(static_cast<int>(x[j]), 0x01010101, sum)
                        : static_cast<int32_t>(__dp4a(x[j], 0x01010101u, static_cast<unsigned>(sum)));
    return sum;
}

template <int MR, bool B_KMAJOR, int OUT>
__global__ void __launch_bounds__(slim::THREADS, 2)
    int8_gemm_slim_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                          const __grid_constant__ SlimParams p, uint32_t idesc, uint32_t idesc_ones) {
    using C = slim::Cfg<MR>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sB = smem;
    uint8_t* sX = smem + C::STAGES * C::B_BYTES;
    uint8_t* sOnes = smem + C::RING;
    uint64_t* bars = reinterpret_cast<uint64_t*>(sOnes + C::ONES_BYTES);
    uint64_t* full = bars;
    uint64_t* empty = bars + C::STAGES;
    uint64_t* tfull = bars + 2 * C::STAGES;
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 2 * C::STAGES + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
    volatile int* ready = reinterpret_cast<volatile int*>(tmem_holder + 2);
    int32_t* col_sum = reinterpret_cast<int32_t*>(reinterpret_cast<uint8_t*>(bars) + 256);  // [128] of this CTA's share
    int32_t* row_sum = col_sum + slim::BN;                                                  // [MR] of this CTA's share
    int32_t* row_all = row_sum + MR;                                                        // [MR] of all of K
    float* row_scale = reinterpret_cast<float*>(row_all + MR);                              // [MR]
    int32_t* row_zero = reinterpret_cast<int32_t*>(row_scale + MR);                         // [MR] zero points of A
    uint32_t* partial = reinterpret_cast<uint32_t*>(smem);                                  // [MR][128], after the MMAs

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int parts = static_cast<int>(gridDim.y), part = static_cast<int>(blockIdx.y);
    const int per_batch = p.tiles * p.row_chunks;
    const int b = static_cast<int>(blockIdx.x) / per_batch, in_batch = static_cast<int>(blockIdx.x) - b * per_batch;
    const int tile = in_batch / p.row_chunks, row0 = (in_batch - tile * p.row_chunks) * MR;  // chunks of a tile are neighbours
    const int kb0 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * part / parts);
    const int kb1 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * (part + 1) / parts);
    const Epilogue& e = p.epi;
    const bool need_col_sums = e.za != nullptr;
    pdl_trigger();

    for (int i = threadIdx.x; i < C::ONES_BYTES / 16; i += blockDim.x)
        reinterpret_cast<uint4*>(sOnes)[i] = make_uint4(0x01010101u, 0x01010101u, 0x01010101u, 0x01010101u);
    fence_proxy_async_smem();  // generic writes -> visible to the tensor cores
    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], p.epi.zb != nullptr ? 5 : 1);  // the MMAs, and the four warps that sum the rows of A
        }
        mbar_init(tfull, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 0 && lane == 0) {
        prefetch_tmap(&tmap_a);
        prefetch_tmap(&tmap_b);
    }
    pdl_wait();  // the preceding grid is done: its outputs are readable and its TMEM is free
    if (warp == 1) {
        tmem_alloc(tmem_holder, C::TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_holder;
    const int ba = p.a_batched ? b : 0, bb = p.b_batched ? b : 0;
    // What the finishing threads need of their column, asked for before B streams.
    const int n = tile * slim::BN + static_cast<int>(threadIdx.x) - 64;
    uint32_t zb = 0, bias = 0;
    float scale = 0.0f, fbias = 0.0f;
    if (warp >= 2 && n < p.n) {
        zb = static_cast<uint32_t>(zp_value(e.zb, e.zb_vector, e.zb_signed, n));
        if (e.int_bias != nullptr) bias = static_cast<uint32_t>(__ldg(e.int_bias + n));
        scale = __ldg(e.scale + (e.scale_vector ? n : 0));
        if (e.float_bias != nullptr) fbias = __ldg(e.float_bias + n);
    }

    int issued = 0;  // by warp 0
    if (warp == 0) {
        const int last = p.withhold && blockIdx.x == 0 && part == 0 ? kb1 - 1 : kb1;
        for (int kb = kb0; kb < last; kb++) {
            const int it = kb - kb0, s = it % C::STAGES;
            if (!mbar_wait_warp(&empty[s], ((it / C::STAGES) & 1) ^ 1, abort_flag, p.wait_limit_ns)) break;
            if (lane == 0) {
                mbar_arrive_expect_tx(&full[s], C::B_BYTES + C::A_BYTES);
                if constexpr (B_KMAJOR)
                    tma_load_3d(sB + s * C::B_BYTES, &tmap_b, &full[s], kb * slim::BK, tile * slim::BN, bb);
                else
                    tma_load_3d(sB + s * C::B_BYTES, &tmap_b, &full[s], tile * slim::BN, kb * slim::BK, bb);
                tma_load_3d(sX + s * C::A_BYTES, &tmap_a, &full[s], kb * slim::BK, row0, ba);
            }
            issued++;
            __syncwarp();
        }
    } else if (warp == 1) {
        bool ok = true;
        for (int kb = kb0; kb < kb1; kb++) {
            const int it = kb - kb0, s = it % C::STAGES;
            ok = mbar_wait_warp(&full[s], (it / C::STAGES) & 1, abort_flag, p.wait_limit_ns);
            if (!ok) break;
            tc_fence_after();
            if (lane == 0) {
                const uint32_t b_addr = smem_u32(sB + s * C::B_BYTES);
                const uint32_t x_addr = smem_u32(sX + s * C::A_BYTES);
                const uint32_t o_addr = smem_u32(sOnes);
#pragma unroll
                for (int kk = 0; kk < slim::BK / 32; kk++) {
                    const uint64_t adesc = B_KMAJOR ? smem_desc_sw128(b_addr + kk * 32, 16, 1024)
                                                    : smem_desc_sw128(b_addr + kk * 32 * 128, C::B_BYTES, 1024);
                    const uint32_t acc = (it != 0 || kk >= C::ACCS) ? 1u : 0u;
                    const uint32_t d = tmem_base + (kk % C::ACCS) * C::ACC_COLS;
                    mma_i8(d, adesc, smem_desc_sw128(x_addr + kk * 32, 16, 1024), idesc, acc);
                    if (need_col_sums)
                        mma_i8(d + MR, adesc, smem_desc_sw128(o_addr + kk * 32, 16, 1024), idesc_ones, acc);
                }
                mma_commit(&empty[s]);
            }
            __syncwarp();
        }
        if (ok && lane == 0) mma_commit(tfull);
        __syncwarp();
    } else {
        const int t = threadIdx.x - 64, w = warp - 2;
        for (int r = t; r < MR && row0 + r < p.m; r += slim::FINISH_THREADS) {
            row_scale[r] = row_scale_of(e, row0 + r);
            row_zero[r] = zp_value(e.za, e.za_vector, e.za_signed, row0 + r);
        }
        if (e.zb != nullptr) {
            // Row sums of A over this CTA's share of K, from the boxes in shared memory (zeros past K and M): LANES threads
            // a row. The order of a row's 16-byte units does not matter, so the swizzle is not undone but used: lanes of
            // different rows read different units.
            constexpr int LANES = slim::FINISH_THREADS / MR, UNITS = 8 / LANES;
            const int r = t / LANES, u0 = (t % LANES) * UNITS;
            int32_t sum = 0;
            for (int kb = kb0; kb < kb1; kb++) {
                const int it = kb - kb0, s = it % C::STAGES;
                if (!mbar_wait_warp(&full[s], (it / C::STAGES) & 1, abort_flag, p.wait_limit_ns)) break;
                const uint4* box = reinterpret_cast<const uint4*>(sX + s * C::A_BYTES + r * slim::BK);
#pragma unroll
                for (int i = 0; i < UNITS; i++) sum = byte_sum(box[(u0 + i) ^ (r & 7)], e.za_signed, sum);
                asm volatile("" ::"r"(sum) : "memory");  // the reads are done before the box is given back
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[s]);
            }
#pragma unroll
            for (int o = 1; o < LANES; o <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
            if (t % LANES == 0) row_sum[r] = sum;
        }
        if (t == 0) *ready = mbar_wait(tfull, 0, abort_flag, p.wait_limit_ns) ? 1 : 0;
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (*ready) {
            tc_fence_after();
            const int col = (warp & 3) * 32 + lane;  // this thread's TMEM lane
            const uint32_t lane_base = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
            const int rows_used = min(MR, p.m - row0);
#pragma unroll 1
            for (int c = 0; c < C::ACC_COLS; c += 16) {
                if (c < MR ? c >= rows_used : !need_col_sums) continue;
                uint32_t r[16];
                tmem_ld_32x32b_x16(lane_base + c, r);
                tmem_ld_wait();
#pragma unroll
                for (int a = 1; a < C::ACCS; a++) {
                    uint32_t x[16];
                    tmem_ld_32x32b_x16(lane_base + a * C::ACC_COLS + c, x);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 16; i++) r[i] += x[i];
                }
                if (c < MR) {
#pragma unroll
                    for (int i = 0; i < 16; i++) partial[(c + i) * slim::BN + col] = r[i];
                } else {
                    col_sum[col] = static_cast<int32_t>(r[0]);
                }
            }
            tc_fence_before();
        }
    }
    __syncwarp();
    cluster_sync_all();  // every CTA's partial sums are in its shared memory
    if (warp == 0 && lane == 0 && *abort_flag) drain_ring(full, C::STAGES, issued);

    if (warp >= 2) {
        const int t = threadIdx.x - 64;
        // Row sums over all of K; a CTA finishes rows part, part + parts, ...
        if (e.zb != nullptr) {
            for (int r = part + t * parts; r < MR && row0 + r < p.m; r += slim::FINISH_THREADS * parts) {
                uint32_t sum = 0;
                for (int q = 0; q < parts; q++) sum += ld_cluster_u32(mapa_shared(smem_u32(row_sum + r), q));
                row_all[r] = static_cast<int32_t>(sum);
            }
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (n < p.n) {
            uint32_t peer[slim::MAX_PARTS];
#pragma unroll
            for (int q = 0; q < slim::MAX_PARTS; q++) peer[q] = mapa_shared(smem_u32(partial + t), q < parts ? q : 0);
            uint32_t csb = 0;
            if (need_col_sums)
                for (int q = 0; q < parts; q++) csb += ld_cluster_u32(mapa_shared(smem_u32(col_sum + t), q));
            const bool biased = e.float_bias != nullptr;
            const int rows_here = min(MR, p.m - row0);
            constexpr int ROWS = MR == 16 ? 4 : 8;  // rows finished together: their loads are in flight together
            const int64_t at = b * e.batch_stride_c + static_cast<int64_t>(row0) * e.ldc + n;
#pragma unroll 1
            for (int r0 = part; r0 < rows_here; r0 += ROWS * parts) {
                float res[ROWS];
                uint32_t s[ROWS];
#pragma unroll
                for (int i = 0; i < ROWS; i++) {  // past the rows, the last one again (not stored)
                    res[i] = e.residual != nullptr
                                 ? residual_at<OUT>(e, at + static_cast<int64_t>(min(r0 + i * parts, rows_here - 1)) * e.ldc)
                                 : 0.0f;
                    s[i] = bias;
                }
#pragma unroll
                for (int q = 0; q < slim::MAX_PARTS; q++) {
                    if (q >= parts) break;
#pragma unroll
                    for (int i = 0; i < ROWS; i++) s[i] += ld_cluster_u32(peer[q] + min(r0 + i * parts, rows_here - 1) * slim::BN * 4);
                }
                float f[ROWS];
#pragma unroll
                for (int i = 0; i < ROWS; i++) {
                    const int r = min(r0 + i * parts, rows_here - 1);
                    const uint32_t za = static_cast<uint32_t>(row_zero[r]);
                    if (e.zb != nullptr) s[i] += zb * (static_cast<uint32_t>(p.k) * za - static_cast<uint32_t>(row_all[r]));
                    if (e.za != nullptr) s[i] -= za * csb;
                    f[i] = scaled_sum(s[i], row_scale[r], scale, biased, fbias);
                }
                activate_all(f, e.activation);
#pragma unroll
                for (int i = 0; i < ROWS; i++) {
                    if (r0 + i * parts >= rows_here) break;
                    const int64_t idx = at + static_cast<int64_t>(r0 + i * parts) * e.ldc;
                    if (e.residual != nullptr) f[i] = __fadd_rn(f[i], res[i]);
                    if constexpr (OUT == OUT_ACT_F16)
                        static_cast<__half*>(e.c)[idx] = __float2half_rn(f[i]);
                    else
                        static_cast<float*>(e.c)[idx] = f[i];
                }
            }
        }
    }
    __syncwarp();
    cluster_sync_all();  // no CTA leaves while another still reads its shared memory
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, C::TMEM_COLS);
    }
    if (threadIdx.x == 0 && *abort_flag) atomicExch(p.error_flag, 1);
}

// ---- host side ------------------------------------------------------------------------------------------------------

static int slim_rows(int m) { return m <= 16 ? 16 : m <= 32 ? 32 : m <= 64 ? 64 : 128; }

// Sets the kernel's shared memory once per device.
template <int MR, class Kernel>
static cudaError_t configure_slim(Kernel kern, std::atomic<uint64_t>& configured) {
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = uint64_t(1) << (dev & 63);
    if (configured.load() & bit) return cudaSuccess;
    const cudaError_t set = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, slim::Cfg<MR>::SMEM_BYTES);
    if (set == cudaSuccess) configured.fetch_or(bit);
    return set;
}

// Clusters of `parts` CTAs that the current device holds at once (a cluster stays within a group of SMs, so this is less
// than its CTA slots over `parts`). One of the kernels of MR stands for all: they hold as much shared memory.
template <int MR>
static int slim_clusters_at_once(int parts) {
    static std::atomic<int> known[64][slim::MAX_PARTS + 1] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    std::atomic<int>& slot = known[dev & 63][parts];
    if (slot.load() != 0) return slot.load();
    static std::atomic<uint64_t> configured{0};
    auto kern = int8_gemm_slim_kernel<MR, true, OUT_ACT_F32>;
    if (configure_slim<MR>(kern, configured) != cudaSuccess) return 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1, static_cast<unsigned>(parts));
    cfg.blockDim = dim3(slim::THREADS);
    cfg.dynamicSmemBytes = slim::Cfg<MR>::SMEM_BYTES;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = static_cast<unsigned>(parts);
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    if (cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg) != cudaSuccess) return 0;
    slot.store(clusters);
    return clusters;
}

static int slim_clusters_at_once(int mr, int parts) {
    switch (mr) {
        case 16: return slim_clusters_at_once<16>(parts);
        case 32: return slim_clusters_at_once<32>(parts);
        case 64: return slim_clusters_at_once<64>(parts);
        default: return slim_clusters_at_once<128>(parts);
    }
}

// The parts of K that a cluster shares, or 0 when the kernel for whole tiles serves better. Up to 64 rows always. From 65
// rows on K needs some length to outweigh the finish, less where whole tiles would need a pass for the byte sums:
// 512 x 2048 x 512 with zero points 23.3 us in whole tiles and 19.4 here, 4096 x 512 x 512 without 17.3 and 19.5. Each 128
// rows read B again (from L2), which pays while whole tiles would leave SMs idle: 256 x 8192 x 8192 55 and 45, 300 x 512 x
// 4096 28.7 and 17.4, 2048 x 256 x 1024 19.3 and 17.3, 2048 x 1024 x 2048 (the edge of the rule) 22.7 and 23.5, with zero
// points 27.6 and 25.6.
// As many parts as still run at once: a cluster left over would wait for a whole pass (5 x 5120 x 5120 with one part more
// 23.4, without 17.4).
int slim_parts(const GemmLaunch& L) {
    if (!out_activated(L.epi.out_kind) || !tc_eligible(L) || L.batch > 65535) return 0;
    const int mr = slim_rows(L.m);
    const int64_t chunks = (L.m + mr - 1) / mr;
    const int64_t tiles = (static_cast<int64_t>(L.n) + slim::BN - 1) / slim::BN * chunks * L.batch;
    const int64_t slots = 2 * static_cast<int64_t>(L.num_sms);  // two CTAs on each SM
    const int64_t k_blocks = (L.k + slim::BK - 1) / slim::BK;
    if (tiles > 0x7FFFFFFF) return 0;
    if (L.m > 64 && k_blocks < (L.epi.za != nullptr || L.epi.zb != nullptr ? 4 : 8)) return 0;
    if (chunks > 1 && 2 * tiles > slots) return 0;
    int64_t parts = std::max<int64_t>(1, std::min<int64_t>({slots / tiles, k_blocks / 2, slim::MAX_PARTS}));
    auto at_once = [&](int64_t size) {  // the query counts one CTA on an SM
        return slots / std::max(1, slim_clusters_at_once(mr, 1)) * slim_clusters_at_once(mr, static_cast<int>(size));
    };
    while (parts > 1 && at_once(parts) < tiles) parts--;
    return static_cast<int>(parts);
}

template <int MR, bool B_KMAJOR, int OUT>
static LaunchFn bind_slim_t(const SlimParams& p, const CUtensorMap& ma, const CUtensorMap& mb, dim3 grid, uint32_t idesc,
                            uint32_t idesc_ones) {
    return [=](cudaStream_t stream) -> cudaError_t {
        using C = slim::Cfg<MR>;
        auto kern = int8_gemm_slim_kernel<MR, B_KMAJOR, OUT>;
        static std::atomic<uint64_t> configured{0};  // devices whose attribute is set
        const cudaError_t e = configure_slim<MR>(kern, configured);
        if (e != cudaSuccess) return e;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = grid;
        cfg.blockDim = dim3(slim::THREADS);
        cfg.dynamicSmemBytes = C::SMEM_BYTES;
        cfg.stream = stream;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 1;
        attr[0].val.clusterDim.y = grid.y;
        attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = pdl_enabled() ? 2 : 1;
        return cudaLaunchKernelEx(&cfg, kern, ma, mb, p, idesc, idesc_ones);
    };
}

template <int MR>
static LaunchFn bind_slim_m(const GemmLaunch& L, const SlimParams& p, const CUtensorMap& ma, const CUtensorMap& mb,
                            dim3 grid) {
    // The MMA's A operand is B (its type, MN-major unless B is stored N x K); its B operand is A (or the ones).
    const uint32_t idesc = idesc_i8(L.b_signed, L.a_signed, !L.trans_b, false, slim::BN, MR);
    const uint32_t ones = idesc_i8(L.b_signed, L.a_signed, !L.trans_b, false, slim::BN, 16);
    const bool f16 = L.epi.out_kind == OUT_ACT_F16;
    if (L.trans_b)
        return f16 ? bind_slim_t<MR, true, OUT_ACT_F16>(p, ma, mb, grid, idesc, ones)
                   : bind_slim_t<MR, true, OUT_ACT_F32>(p, ma, mb, grid, idesc, ones);
    return f16 ? bind_slim_t<MR, false, OUT_ACT_F16>(p, ma, mb, grid, idesc, ones)
               : bind_slim_t<MR, false, OUT_ACT_F32>(p, ma, mb, grid, idesc, ones);
}

LaunchFn prepare_gemm_slim(const GemmLaunch& L, int parts, uint64_t self_test_ns, cudaError_t* err) {
    *err = cudaErrorInvalidValue;
    const int mr = slim_rows(L.m);
    const int ba = (L.batch > 1 && L.stride_a != 0) ? L.batch : 1;
    const int bb = (L.batch > 1 && L.stride_b != 0) ? L.batch : 1;
    CUtensorMap ma, mb;
    const uint64_t sa = ba > 1 ? uint64_t(L.stride_a) : (uint64_t(L.lda) * L.m + 15) & ~uint64_t(15);
    if (!make_tensor_map_u8(&ma, L.a, L.k, L.m, ba, L.lda, sa, slim::BK, mr)) return nullptr;
    const uint64_t rows_b = L.trans_b ? L.n : L.k;
    const uint64_t sb = bb > 1 ? uint64_t(L.stride_b) : (uint64_t(L.ldb) * rows_b + 15) & ~uint64_t(15);
    const bool ok = L.trans_b ? make_tensor_map_u8(&mb, L.b, L.k, L.n, bb, L.ldb, sb, slim::BK, slim::BN)
                              : make_tensor_map_u8(&mb, L.b, L.n, L.k, bb, L.ldb, sb, slim::BN, slim::BK);
    if (!ok) return nullptr;
    *err = cudaSuccess;
    SlimParams p = {};
    p.m = L.m;
    p.n = L.n;
    p.k = L.k;
    p.k_blocks = (L.k + slim::BK - 1) / slim::BK;
    p.tiles = (L.n + slim::BN - 1) / slim::BN;
    p.row_chunks = (L.m + mr - 1) / mr;
    p.a_batched = ba > 1;
    p.b_batched = bb > 1;
    p.epi = L.epi;
    p.error_flag = L.error_flag;
    p.wait_limit_ns = self_test_ns != 0 ? self_test_ns : OG_WAIT_LIMIT_NS;
    p.withhold = self_test_ns != 0;
    const dim3 grid(static_cast<unsigned>(p.tiles * p.row_chunks * L.batch), static_cast<unsigned>(parts));
    switch (mr) {
        case 16: return bind_slim_m<16>(L, p, ma, mb, grid);
        case 32: return bind_slim_m<32>(L, p, ma, mb, grid);
        case 64: return bind_slim_m<64>(L, p, ma, mb, grid);
        default: return bind_slim_m<128>(L, p, ma, mb, grid);
    }
}

}  // namespace og
