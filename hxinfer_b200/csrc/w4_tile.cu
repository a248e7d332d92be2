// w4_tile.cu — the 4-bit linear product on the 5th-generation tensor cores, for
// the calls with too many tokens for mma.sync (layout and formula: w4_linear.cu).
//
//   y[t][o] = sum_g s[o][g] * ( sum_{k in g} (c[o][k] - z[o][g]) x[t][k] ) + b[o]
//
// A tile is 128 outputs (M, eight of the layout's row tiles) by N tokens; its
// inputs come in units of 128.  For every unit the codes are turned into c - z,
// exact in fp16, and written to shared memory as the A operand; x comes as the
// B operand by TMA.  The products of one group of inputs accumulate in fp32 in
// tensor memory, in a buffer of their own, from where the scale warps take the
// sums, multiply them by the row's scale and add them up in fp32 registers: as
// on the other paths nothing is rounded before y.
//
// Roles of a CTA's warps: scale warps (a thread holds one output's sums of 64
// tokens), 8 conversion warps (one row tile each), and one warp each for the
// copies of weights, those of x, and the MMAs.  They meet only at mbarriers, so
// copies, conversion, products and scales of different units overlap.
//
// A cluster of CTAs shares a tile when there are too few tiles for all SMs: its
// CTAs take a part of the inputs each, leave their sums in shared memory, and
// each adds up (in the order of the CTAs) and stores a part of the tokens.
//
// What bounds it: a unit takes 0.7 us, 0.43 us of it the roles' hand-overs (what
// is left with the copies, the conversion and all but one MMA taken out), 0.15
// us the conversion and the rest the products, nearly whatever the number of
// tokens.  So tiles are wide, 64 or 128 tokens, and 32 tokens or fewer stay on
// mma.sync (32 x 4096 x 28672: 41 us there, 51 here with 32-token tiles; 17 x
// 11008 x 4099: 13 and 28; 33 x 4096 x 14336: 45 and 28).  Measured: 64 x 4096
// x 14336 29 us, 128 x 4096 x 14336 32 us (470 Tflop/s), 512 x 4096 x 4096 31 us
// (550), 1024 x 4096 x 14336 187 us (640), in a graph; w4_linear_kernel took 47,
// 85, 109 and 531.
#include <algorithm>
#include <atomic>

#include "hx_tcgen05.cuh"
#include "hx_w4.cuh"

namespace hx {

constexpr int kWtConvertWarps = 8;
constexpr int kWtRows = 128;
constexpr int kWtRegion = kWtRows * 128;  // 128 rows x 64 fp16, 128-byte swizzle
// What a tile costs a CTA besides its units, and what sharing it adds, in units.
constexpr int kWtTileCost = 2, kWtSplitCost = 2;

template <int N, int GROUP, bool ZEROS>
struct W4Tile {
    static constexpr int kGroups = kW4Unit / GROUP;
    static constexpr int kCodes = kW4Rows * kW4Unit / 2;
    static constexpr int kRecord = kCodes + kGroups * kW4Rows * (ZEROS ? 3 : 2);
    static constexpr int kScaleWarps = N / 16;     // 32 outputs by 64 tokens each
    static constexpr int kWeightWarp = kScaleWarps + kWtConvertWarps, kInputWarp = kWeightWarp + 1;
    static constexpr int kMmaWarp = kInputWarp + 1, kThreads = 32 * (kMmaWarp + 1);
    static constexpr int kStages = 2;              // units of A
    static constexpr int kInputs = N > 64 ? 2 : 3; // of x
    static constexpr int kSlots = 6;               // of records
    static constexpr int kSums = 4;                // buffers of N columns in tensor memory
    static constexpr int kMaxSplit = N > 64 ? 1 : 8;
    static constexpr int kColumns = N * kSums;
    // Units of scales.  Unit n's are written once the MMAs of unit
    // n - 1 - kStages have finished, which waited for the sums of the groups
    // kSums before them: the scales of unit n - kScales have been used.
    static constexpr int kScales = 1 + kStages + kSums / kGroups;

    struct Smem {
        uint8_t a[kStages][2][kWtRegion];        // [64-input half]
        uint8_t x[kInputs][2][N * 128];
        float part[kMaxSplit > 1 ? N : 1][kWtRows];  // sums that the cluster adds up
        __half scale[kScales][kGroups][kWtRows];
        uint8_t raw[kSlots][kWtRows / kW4Rows][kRecord];
        uint64_t raw_full[kSlots], raw_empty[kSlots];
        uint64_t x_full[kInputs], x_empty[kInputs];
        uint64_t a_full[kStages], a_empty[kStages];
        uint64_t sum_full[kSums], sum_empty[kSums];
        uint64_t part_full, part_free, mma_idle;
        uint32_t tmem_base;
        int abort_flag;
    };
};

struct W4Split {
    int split, clusters;   // CTAs that share a tile, clusters launched
    int groups;            // of N tokens
    int64_t items;         // tiles
};

__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ uint32_t cluster_addr(const void* p, int rank)
{
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}

__device__ __forceinline__ void cluster_arrive(uint64_t* bar, int rank)
{
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr(bar, rank)) : "memory");
}

__device__ __forceinline__ float cluster_load(const float* p, int rank)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr(p, rank)) : "memory");
    return v;
}

// 32 codes of two rows (low: nibbles 0, 2, 4, 6; high: 1, 3, 5, 7) of one word.
__device__ __forceinline__ void w4_convert(uint32_t w, uint32_t lo_off, uint32_t hi_off, uint32_t* lo, uint32_t* hi)
{
    const uint32_t e = w >> 8;
    lo[0] = h2_sub(lop_and_or(w, 0x000f000fu, 0x64006400u), lo_off);
    hi[0] = h2_sub(lop_and_or(w, 0x00f000f0u, 0x54005400u), hi_off);
    lo[1] = h2_sub(lop_and_or(e, 0x000f000fu, 0x64006400u), lo_off);
    hi[1] = h2_sub(lop_and_or(e, 0x00f000f0u, 0x54005400u), hi_off);
}

template <int N, int GROUP, bool ZEROS>
__global__ void __launch_bounds__(W4Tile<N, GROUP, ZEROS>::kThreads, 1)
    w4_tile_kernel(const __grid_constant__ CUtensorMap tm_x, const W4Params p, const W4Split w)
{
    using Tile = W4Tile<N, GROUP, ZEROS>;
    constexpr int kStages = Tile::kStages, kInputs = Tile::kInputs, kSlots = Tile::kSlots, kSums = Tile::kSums, kRecord = Tile::kRecord;
    extern __shared__ uint8_t smem_raw[];
    auto& sm = *reinterpret_cast<typename Tile::Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x % w.split, cluster = blockIdx.x / w.split;
    if (threadIdx.x == 0) {
        prefetch_tensormap(&tm_x);
        for (int i = 0; i < kSlots; ++i) {
            mbar_init(&sm.raw_full[i], 1);
            mbar_init(&sm.raw_empty[i], kWtConvertWarps);
        }
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&sm.a_full[i], kWtConvertWarps);
            mbar_init(&sm.a_empty[i], 1);
        }
        for (int i = 0; i < kInputs; ++i) {
            mbar_init(&sm.x_full[i], 1);
            mbar_init(&sm.x_empty[i], 1);
        }
        for (int i = 0; i < kSums; ++i) {
            mbar_init(&sm.sum_full[i], 2);
            mbar_init(&sm.sum_empty[i], Tile::kScaleWarps);
        }
        mbar_init(&sm.part_full, Tile::kScaleWarps * w.split);
        mbar_init(&sm.part_free, Tile::kScaleWarps * w.split);
        mbar_init(&sm.mma_idle, 1);
        sm.abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == Tile::kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem_base)),
                     "n"(Tile::kColumns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // the others' barriers are ready
    tc_fence_after();
    pdl_wait();  // x, and perhaps the weight, come from earlier kernels on the stream
    pdl_trigger();
    const uint32_t tmem = sm.tmem_base;
    const int u0 = (int)((int64_t)p.s.units * rank / w.split), u1 = (int)((int64_t)p.s.units * (rank + 1) / w.split);
    // a bounded wait; false ends the role
    auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait_or_abort(&sm.abort_flag, bar, parity, p.status); };
    // the same for a whole warp
    auto warp_wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
    // tile `item`: its first row tile, how many exist, its first token
    auto tile0 = [&](int64_t item) { return item / w.groups * (kWtRows / kW4Rows); };
    auto live = [&](int64_t item) { return (int)min((int64_t)(kWtRows / kW4Rows), p.s.tiles - tile0(item)); };
    auto token0 = [&](int64_t item) { return (int)(item % w.groups) * N; };

    if (warp == Tile::kWeightWarp) {
        // a lane per row tile issues its copy
        const uint64_t pol = l2_evict_first_policy();
        const int64_t tile_bytes = (int64_t)p.s.units * kRecord;
        int n = 0;  // units so far: the rings' phases
        bool ok = true;
        for (int64_t item = cluster; ok && item < w.items; item += w.clusters) {
            const char* src = p.packed + (tile0(item) + lane) * tile_bytes + (int64_t)u0 * kRecord;
            const int tiles = live(item);
            for (int u = u0; u < u1; ++u, ++n, src += kRecord) {
                const int slot = n % kSlots;
                ok = n < kSlots || warp_wait(&sm.raw_empty[slot], (n / kSlots - 1) & 1);
                if (!ok) break;
                if (lane == 0) mbar_arrive_expect_tx(&sm.raw_full[slot], tiles * kRecord);
                __syncwarp();
                if (lane < tiles) bulk_load(sm.raw[slot][lane], src, kRecord, &sm.raw_full[slot], pol);
            }
        }
        // copies in flight land before the CTA ends (bounded)
        for (int i = max(0, n - kSlots); i < n; ++i) mbar_wait(&sm.raw_full[i % kSlots], (i / kSlots) & 1);
    } else if (warp == Tile::kInputWarp) {
        if (lane == 0) {
            const uint64_t pol = l2_evict_last_policy();  // every tile reads x
            int n = 0;
            bool ok = true;
            for (int64_t item = cluster; ok && item < w.items; item += w.clusters) {
                for (int u = u0; u < u1; ++u, ++n) {
                    const int st = n % kInputs;
                    ok = n < kInputs || wait(&sm.x_empty[st], (n / kInputs - 1) & 1);
                    if (!ok) break;
                    mbar_arrive_expect_tx(&sm.x_full[st], N * 256);  // what lies outside of x is filled with zeros
                    tma_load_2d(sm.x[st][0], &tm_x, u * kW4Unit, token0(item), &sm.x_full[st], pol);
                    tma_load_2d(sm.x[st][1], &tm_x, u * kW4Unit + 64, token0(item), &sm.x_full[st], pol);
                }
            }
            for (int i = max(0, n - kInputs); i < n; ++i) mbar_wait(&sm.x_full[i % kInputs], (i / kInputs) & 1);
        }
    } else if (warp == Tile::kMmaWarp) {
        // the whole warp waits and one lane issues: descriptors stay in uniform registers
        const uint32_t idesc = umma_idesc(false, N);
        const uint64_t a_desc = umma_desc(smem_u32(sm.a[0][0]), 16, 1024);
        const uint64_t x_desc = umma_desc(smem_u32(sm.x[0][0]), 16, 1024);
        int n = 0, d = 0;  // units and groups so far
        bool ok = true;
        for (int64_t item = cluster; ok && item < w.items; item += w.clusters) {
            for (int u = u0; ok && u < u1; ++u, ++n) {
                const int st = n % kStages, in = n % kInputs;
                ok = warp_wait(&sm.x_full[in], (n / kInputs) & 1) && warp_wait(&sm.a_full[st], (n / kStages) & 1);
                if (!ok) break;
                const uint64_t ad = a_desc + (uint64_t)st * (2 * kWtRegion >> 4);
                const uint64_t xd = x_desc + (uint64_t)in * (N * 256 >> 4);
#pragma unroll
                for (int gr = 0; gr < Tile::kGroups; ++gr, ++d) {
                    const int b = d % kSums;
                    ok = d < kSums || warp_wait(&sm.sum_empty[b], (d / kSums - 1) & 1);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int kk = gr * GROUP / 16; kk < (gr + 1) * GROUP / 16; ++kk)
                            umma_f16(tmem + b * N, ad + (uint64_t)(((kk >> 2) * kWtRegion + (kk & 3) * 32) >> 4),
                                     xd + (uint64_t)(((kk >> 2) * (N * 128) + (kk & 3) * 32) >> 4), idesc,
                                     kk > gr * GROUP / 16);
                        umma_commit(&sm.sum_full[b]);
                        mbar_arrive(&sm.sum_full[b]);  // hands the conversion's scales on
                    }
                }
                if (ok && elect_one()) {
                    umma_commit(&sm.a_empty[st]);
                    umma_commit(&sm.x_empty[in]);
                }
            }
        }
        if (elect_one()) umma_commit(&sm.mma_idle);  // every MMA has finished before the CTA ends
        if (!mbar_wait(&sm.mma_idle, 0)) record_status(p.status, HX_ERR_TIMEOUT);
    } else if (warp >= Tile::kScaleWarps) {
        // conversion: row tile `t` of every unit
        const int t = warp - Tile::kScaleWarps, g = lane >> 2, t4 = lane & 3;
        const bool odd = g & 1;
        // row g (and, 1,024 bytes on, g + 8) of the tile; chunk c of a row lies at c ^ (row % 8)
        const uint32_t row = (kW4Rows * t + g) * 128, ch0 = (t4 ^ g) << 4, ch1 = ch0 ^ 64;
        int n = 0;
        bool ok = true;
        for (int64_t item = cluster; ok && item < w.items; item += w.clusters) {
            const bool mine = t < live(item);
            for (int u = u0; u < u1; ++u, ++n) {
                const int slot = n % kSlots, st = n % kStages;
                ok = warp_wait(&sm.raw_full[slot], (n / kSlots) & 1);
                if (!ok) break;
                uint4 c[2];
                uint32_t zz[ZEROS ? Tile::kGroups : 1];
                if (mine) {
                    const uint8_t* rec = sm.raw[slot][t];
                    c[0] = *reinterpret_cast<const uint4*>(rec + 16 * lane);
                    c[1] = *reinterpret_cast<const uint4*>(rec + 512 + 16 * lane);
                    // two rows' scales a lane, as they lie: rows g and g + 8
                    if (lane < 8 * Tile::kGroups)
                        *reinterpret_cast<__half2*>(&sm.scale[n % Tile::kScales][lane / 8][kW4Rows * t + 2 * (lane % 8)]) =
                            *reinterpret_cast<const __half2*>(rec + Tile::kCodes + 4 * lane);
                    if constexpr (ZEROS)
#pragma unroll
                        for (int gr = 0; gr < Tile::kGroups; ++gr)
                            zz[gr] = *reinterpret_cast<const uint16_t*>(rec + Tile::kCodes + Tile::kGroups * kW4Rows * 2 +
                                                                        gr * kW4Rows + 2 * g);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.raw_empty[slot]);
                ok = n < kStages || warp_wait(&sm.a_empty[st], (n / kStages - 1) & 1);
                if (!ok) break;
                if (mine) {
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        // Odd rows store the second half first: the 8 lanes of a
                        // 128-byte store then reach every bank once.
                        uint8_t* dst = sm.a[st][b] + row;
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int q0 = 2 * b + i, q1 = 2 * b + 1 - i;  // even rows' quarter, odd rows'
                            const uint32_t w0 = i ? (odd ? c[b].x : c[b].z) : (odd ? c[b].z : c[b].x);
                            const uint32_t w1 = i ? (odd ? c[b].y : c[b].w) : (odd ? c[b].w : c[b].y);
                            uint32_t lo_off = 0x64086408u, hi_off = 0x54805480u;  // 1024 + z, 64 + z
                            if constexpr (ZEROS) {
                                const uint32_t ze = zz[q0 * 32 / GROUP], zo = zz[q1 * 32 / GROUP], z = odd ? zo : ze;
                                lo_off = (0x6400u + (z & 0xff)) * 0x10001u;
                                hi_off = (0x5400u + (z >> 8 << 4)) * 0x10001u;
                            }
                            uint32_t lo[4], hi[4];
                            w4_convert(w0, lo_off, hi_off, lo, hi);
                            w4_convert(w1, lo_off, hi_off, lo + 2, hi + 2);
                            const uint32_t at = (i != 0) != odd ? ch1 : ch0;
                            *reinterpret_cast<uint4*>(dst + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                            *reinterpret_cast<uint4*>(dst + 1024 + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        }
                    }
                    fence_proxy_async_smem();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.a_full[st]);
            }
        }
    } else {
        // scales: output `r` of the tile, 64 tokens from `col` on (a warp reaches the
        // tensor-memory lanes of its quarter)
        const int quarter = warp % 4, col = warp / 4 * 64, r = 32 * quarter + lane;
        const uint32_t taddr = tmem + ((uint32_t)(32 * quarter) << 16) + col;
        const int sr = r / kW4Rows * kW4Rows + 2 * (r % 8) + r / 8 % 2;  // its scale's place
        constexpr int kLoad = N > 64 ? 8 : 32;  // columns at a time: registers
        int n = 0, d = 0, done = 0;
        bool ok = true;
        for (int64_t item = cluster; ok && item < w.items; item += w.clusters, ++done) {
            float acc[64];
#pragma unroll
            for (int i = 0; i < 64; ++i) acc[i] = 0.f;
            for (int u = u0; ok && u < u1; ++u, ++n) {
#pragma unroll 1
                for (int gr = 0; gr < Tile::kGroups; ++gr, ++d) {
                    const int b = d % kSums;
                    ok = warp_wait(&sm.sum_full[b], (d / kSums) & 1);
                    if (!ok) break;
                    tc_fence_after();
                    const float s = __half2float(sm.scale[n % Tile::kScales][gr][sr]);
#pragma unroll
                    for (int c = 0; c < 64; c += kLoad) {
                        float v[kLoad];
                        if constexpr (kLoad == 8) tmem_ld8(taddr + b * N + c, v);
                        else tmem_ld32(taddr + b * N + c, v);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < kLoad; ++i) acc[c + i] = fmaf(s, v[i], acc[c + i]);
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sm.sum_empty[b]);
                }
            }
            if (!ok) break;
            const int64_t out = tile0(item) * kW4Rows + r;
            const int t0 = token0(item);
            const float bias = p.bias && out < p.s.out ? __half2float(p.bias[out]) : 0.f;
            auto store = [&](int i, float y) {
                if (t0 + i >= p.n || out >= p.s.out) return;
                const int64_t at = (int64_t)(t0 + i) * p.s.out + out;
                if (p.y_f32) static_cast<float*>(p.y)[at] = y + bias;
                else static_cast<__half*>(p.y)[at] = __float2half_rn(y + bias);
            };
            if (w.split == 1) {
#pragma unroll
                for (int i = 0; i < 64; ++i) store(col + i, acc[i]);
                continue;
            }
            if constexpr (Tile::kMaxSplit > 1) {
                // the others have read the last tile's sums
                if (done > 0) ok = warp_wait(&sm.part_free, (done - 1) & 1);
                if (!ok) break;
                asm volatile("fence.acq_rel.cluster;" ::: "memory");
#pragma unroll
                for (int i = 0; i < N; ++i) sm.part[i][r] = acc[i];
                __syncwarp();
                if (lane < w.split) cluster_arrive(&sm.part_full, lane);
                ok = warp_wait(&sm.part_full, done & 1);
                if (!ok) break;
                asm volatile("fence.acq_rel.cluster;" ::: "memory");
                const int tok0 = N * rank / w.split, tok1 = N * (rank + 1) / w.split;  // this CTA stores
                for (int i = tok0; i < tok1 && t0 + i < p.n; ++i) {
                    float y = 0.f;
                    for (int c = 0; c < w.split; ++c) y += cluster_load(&sm.part[i][r], c);
                    store(i, y);
                }
                __syncwarp();
                if (lane < w.split) cluster_arrive(&sm.part_free, lane);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == Tile::kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(Tile::kColumns) : "memory");
    }
    cluster_sync();  // no CTA ends while another reads its sums
}

template <int N, int GROUP, bool ZEROS>
static int launch_tile(const W4Params& p, cudaStream_t stream)
{
    using Tile = W4Tile<N, GROUP, ZEROS>;
    auto kernel = w4_tile_kernel<N, GROUP, ZEROS>;
    const size_t smem = sizeof(typename Tile::Smem) + 1024;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(Tile::kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    auto set_split = [&](int split, int clusters) {
        attr[1].val.clusterDim.x = split;
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.gridDim = dim3(split * clusters);
    };
    // clusters of 1, 2, 4 and 8 CTAs that run at once; per device, asked again on ordinals past 63
    static std::atomic<int> room[64][4];
    int dev = 0, n[4];
    HX_CUDA_TRY(cudaGetDevice(&dev));
    const bool kept = dev >= 0 && dev < 64;
    if (kept && room[dev][3].load(std::memory_order_acquire) > 0) {
        for (int i = 0; i < 4; ++i) n[i] = room[dev][i].load(std::memory_order_relaxed);
    } else {
        HX_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        for (int i = 0; i < 4; ++i) {
            set_split(1 << i, num_sms() >> i);
            HX_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n[i], kernel, &cfg));
            n[i] = std::max(1, std::min(n[i], num_sms() >> i));
        }
        if (kept)
            for (int i = 0; i < 4; ++i) room[dev][i].store(n[i], i == 3 ? std::memory_order_release : std::memory_order_relaxed);
    }
    W4Split w{};
    w.groups = (p.n + N - 1) / N;
    w.items = (int64_t)((p.s.tiles + kWtRows / kW4Rows - 1) / (kWtRows / kW4Rows)) * w.groups;
    // The split whose busiest CTA has the least to do, in units: its tiles, each
    // with its part of the inputs and what a tile costs besides.
    int64_t best = INT64_MAX;
    for (int i = 0; i < 4 && 1 << i <= std::min(p.s.units, Tile::kMaxSplit); ++i) {
        const int64_t rounds = (w.items + n[i] - 1) / n[i];
        const int64_t cost = rounds * (((p.s.units + (1 << i) - 1) >> i) + kWtTileCost + (i ? kWtSplitCost : 0));
        if (cost >= best) continue;
        best = cost;
        w.split = 1 << i;
        w.clusters = (int)std::min<int64_t>(w.items, n[i]);
    }
    CUtensorMap tm_x;
    const uint64_t dims[2] = {(uint64_t)p.s.in, (uint64_t)p.n}, strides[1] = {(uint64_t)p.s.in * 2};
    const uint32_t box[2] = {64, N};
    if (int rc = encode_fp16_map(&tm_x, 2, p.x, dims, strides, box)) return rc;
    set_split(w.split, w.clusters);
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, tm_x, p, w);
    if (e != cudaSuccess) return cuda_fail(e, "w4_tile_kernel launch");
    return check_launch("w4_tile_kernel");
}

template <int N>
static int launch_tile_group(const W4Params& p, bool zeros, cudaStream_t s)
{
    if (p.s.group == 32) return zeros ? launch_tile<N, 32, true>(p, s) : launch_tile<N, 32, false>(p, s);
    if (p.s.group == 64) return zeros ? launch_tile<N, 64, true>(p, s) : launch_tile<N, 64, false>(p, s);
    return zeros ? launch_tile<N, 128, true>(p, s) : launch_tile<N, 128, false>(p, s);
}

// 128 tokens a tile where that still gives three SMs in four a tile (512 x 4096
// x 4096: 33.4 us, 57.3 with 64); else 64, which clusters can share.
int launch_w4_tile(const W4Params& p, bool zeros, cudaStream_t stream)
{
    const int64_t wide = (int64_t)((p.s.tiles + kWtRows / kW4Rows - 1) / (kWtRows / kW4Rows)) * ((p.n + 127) / 128);
    if (p.n > 64 && 4 * wide >= 3 * num_sms()) return launch_tile_group<128>(p, zeros, stream);
    return launch_tile_group<64>(p, zeros, stream);
}

}  // namespace hx
