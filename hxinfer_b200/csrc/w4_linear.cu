// w4_linear.cu — projections of a few tokens with 4-bit weights: quantisation,
// layout and the product y = W x + b.  Beside hx_qkv_rope_append (fp16
// weights): a decode step reads every weight once, so a quarter of the bytes
// is up to a quarter of the time.  The reference engine has no counterpart
// (its linear layers are cuBLAS GEMVs over fp16/fp32, matmul_cuda.cu:106-189).
//
//   y[t][o] = sum_g s[o][g] * ( sum_{k in g} (c[o][k] - z[o][g]) x[t][k] ) + b[o]
//
// c - z is a small integer, exact in fp16, so the inner sum is a product of
// fp16 values on the tensor cores with fp32 accumulation, and the scale is
// applied to it in fp32: nothing is rounded before y.
//
// Layout of a packed weight (rows padded to 16, inputs to 128): for every tile
// of 16 rows, for every unit of 128 inputs, one record of
//   codes  [2 blocks of 64 inputs][32 lanes][4 words]
//   scales [groups][8][2] fp16, rows g and g + 8 of the tile in a pair
//   zeros  [groups][8][2] bytes, likewise (only with zero points)
// so that a warp's share of a row tile is one stream of memory, fetched by
// bulk copies into a ring of the warp's own; nothing but x comes by way of
// registers, and registers are left for enough warps to hide the arithmetic.
// The codes of a block are, one word a lane, the A operand of four m16n8k16
// products, 16 rows by 64 inputs.  Which input stands at which k of the product
// is free as long as both operands agree, so lane (g, t4) holds for k step s
// the inputs
//   64 b + 32 (s / 2) + 8 t4 + 4 (s % 2) + {0, 1, 2, 3}
// of rows g and g + 8: a step stays inside one group of 32, and the lane's x
// operand is two contiguous 16-byte chunks, read from global memory without
// staging.  Word s holds those eight codes as nibbles (0, 4) = row g, inputs
// 0 and 1; (1, 5) = row g + 8, inputs 0 and 1; (2, 6) and (3, 7) = inputs 2
// and 3: one mask each turns a nibble pair into two fp16, 1024 + c for the even
// ones and 64 + c for the odd ones (a nibble 4 bits up, under a smaller
// exponent), and one subtraction into c - z.
#include <algorithm>

#include "hx_common.cuh"

namespace hx {

constexpr int kW4Rows = 16;
constexpr int kW4Unit = 128;   // inputs one warp takes at a time: two 64-input blocks
constexpr int kW4MaxWarps = 16;

struct W4Shape {
    int out, in, group;
    int tiles, units;           // of the padded weight
    int record;                 // bytes of a unit of a row tile
    size_t bytes;
};

// False when the sizes are not supported.
static bool w4_shape(int out, int in, int group, bool zeros, W4Shape& s)
{
    if (out < 1 || in < 1 || (group != 32 && group != 64 && group != 128) || in % group) return false;
    s.out = out;
    s.in = in;
    s.group = group;
    s.tiles = out / kW4Rows + (out % kW4Rows != 0);
    s.units = in / kW4Unit + (in % kW4Unit != 0);
    s.record = kW4Rows * kW4Unit / 2 + kW4Unit / group * kW4Rows * (zeros ? 3 : 2);
    s.bytes = (size_t)s.tiles * s.units * s.record;
    return true;
}

// One CTA of 256 threads per record, one thread per word of codes, then one
// per scale and zero point (padding is code 0 under a scale of 0).
__global__ void w4_pack_kernel(const uint8_t* __restrict__ codes, const __half* __restrict__ scales,
                               const uint8_t* __restrict__ zeros, W4Shape s, char* __restrict__ packed)
{
    const int64_t records = (int64_t)s.tiles * s.units;
    const int per = kW4Unit / s.group, in_groups = s.in / s.group;
    for (int64_t rec = blockIdx.x; rec < records; rec += gridDim.x) {
        char* dst = packed + rec * s.record;
        const int64_t row0 = rec / s.units * kW4Rows;
        const int unit = (int)(rec % s.units), i = threadIdx.x;
        const int step = i & 3, lane = (i >> 2) & 31, g = lane >> 2, t4 = lane & 3;
        const int k0 = unit * kW4Unit + 64 * (i >> 7) + 32 * (step / 2) + 8 * t4 + 4 * (step % 2);
        uint32_t w = 0;
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            // nibble n < 4: (row half n & 1, input 2 (n / 2)); n >= 4: the input after it
            const int64_t row = row0 + g + 8 * (n & 1);
            const int k = k0 + 2 * ((n & 3) >> 1) + (n >> 2);
            const uint32_t c = row < s.out && k < s.in ? codes[row * s.in + k] & 15u : 0u;
            w |= c << (4 * n);
        }
        reinterpret_cast<uint32_t*>(dst)[i] = w;
        if (i < per * kW4Rows) {
            const int64_t row = row0 + ((i & 15) >> 1) + 8 * (i & 1);
            const int grp = unit * per + (i >> 4);
            const bool in = row < s.out && grp < in_groups;
            char* sc = dst + kW4Rows * kW4Unit / 2;
            reinterpret_cast<__half*>(sc)[i] = in ? scales[row * in_groups + grp] : __float2half(0.f);
            if (zeros) reinterpret_cast<uint8_t*>(sc + per * kW4Rows * 2)[i] = in ? zeros[row * in_groups + grp] & 15 : 0;
        }
    }
}

// One warp per (row, group).  w and s have 11-bit significands, so the fp32
// quotient is never rounded onto a half-way point it is not on, and the codes
// are those of exact arithmetic.
__global__ void w4_quantize_kernel(const __half* __restrict__ w, int64_t groups, int group,
                                   uint8_t* __restrict__ codes, __half* __restrict__ scales)
{
    const int lane = threadIdx.x & 31;
    for (int64_t i = (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32; i < groups;
         i += (int64_t)gridDim.x * (blockDim.x / 32)) {
        float x[4], mx = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[e] = 32 * e < group ? __half2float(w[i * group + 32 * e + lane]) : 0.f;
            mx = fmaxf(mx, fabsf(x[e]));
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const __half sh = __float2half_rn(mx / 7.f);
        const float s = __half2float(sh);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (32 * e >= group) break;
            // a scale that fp16 rounded far down (subnormal) leaves |w / s| above 7
            const float c = s > 0.f ? fminf(fmaxf(rintf(x[e] / s), -8.f), 7.f) : 0.f;
            codes[i * group + 32 * e + lane] = (uint8_t)((int)c + 8);
        }
        if (lane == 0) scales[i] = sh;
    }
}

__device__ __forceinline__ uint32_t lop_and_or(uint32_t a, uint32_t mask, uint32_t orv)
{
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(a), "r"(mask), "r"(orv));  // (a & mask) | orv
    return d;
}

__device__ __forceinline__ uint32_t h2_sub(uint32_t a, uint32_t b)
{
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// Untiled bulk copy global -> shared (16-byte aligned, a multiple of 16 bytes).
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar, uint64_t policy)
{
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(
            smem_u32(dst)),
        "l"(src), "r"(bytes), "r"(smem_u32(bar)), "l"(policy)
        : "memory");
}

// D = A(16x16 fp16, row) * B(16x8 fp16, col): the first product of a sum.
__device__ __forceinline__ void mma_16816_first(float* d, const uint32_t* a, uint32_t b0, uint32_t b1)
{
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

struct W4Params {
    W4Shape s;
    const __half* x;
    const char* packed;
    const __half* bias;
    void* y;
    int n, y_f32;
    int* status;
};

// One CTA per (RT row tiles, token group of 8 NT).  Its warps take 128-input
// units in turn, U at a time, for all RT tiles, and add their partial sums in
// shared memory in a fixed order.  RT tiles share the x operand, which for
// several tokens is more data than one tile's weights.
template <int NT, int RT, int U, int SLOTS, int GROUP, bool ZEROS>
__global__ void __launch_bounds__(kW4MaxWarps * 32) w4_linear_kernel(const W4Params p)
{
    constexpr int kGroups = kW4Unit / GROUP;  // groups in a unit
    constexpr int kPer = GROUP / 32;          // 32-input quarters in a group
    constexpr int kCodes = kW4Rows * kW4Unit / 2, kScales = kGroups * kW4Rows * 2;
    constexpr int kRecord = kCodes + kScales + (ZEROS ? kGroups * kW4Rows : 0);
    constexpr int kSlot = RT * U * kRecord;   // bytes
    constexpr int kCols = 8 * NT + 1;         // a warp's partial sums [16 RT][8 NT + 1] take its ring's place
    static_assert(SLOTS * kSlot >= RT * 16 * kCols * 4, "partial sums");
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ uint64_t bars[kW4MaxWarps][SLOTS];
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int64_t tile0 = (int64_t)blockIdx.x * RT;
    const int t0 = blockIdx.y * 8 * NT;
    uint8_t* ring = smem + (size_t)warp * SLOTS * kSlot;
    uint64_t* full = bars[warp];
    const int rt = (int)min((int64_t)RT, p.s.tiles - tile0);  // tiles that exist
    const int chunks = (p.s.units + U - 1) / U;               // of U units; this warp's: warp, warp + warps, ...
    const uint64_t pol = l2_evict_first_policy();
    if (lane == 0) {
        for (int i = 0; i < SLOTS; ++i) mbar_init(&full[i], 1);
        fence_mbar_init();
    }
    const int64_t tile_bytes = (int64_t)p.s.units * kRecord;
    const char* src = p.packed + tile0 * tile_bytes + warp * U * kRecord;  // of the next chunk to copy
    const uint32_t last_bytes = (p.s.units - (chunks - 1) * U) * kRecord;
    auto issue = [&](int c, int slot) {  // lane 0
        const uint32_t n = U == 1 || c + 1 < chunks ? U * kRecord : last_bytes;
        uint8_t* dst = ring + slot * kSlot;
        mbar_arrive_expect_tx(&full[slot], RT == 1 ? n : n * rt);
#pragma unroll
        for (int r = 0; r < RT; ++r)
            if (RT == 1 || r < rt) bulk_load(dst + r * U * kRecord, src + r * tile_bytes, n, &full[slot], pol);
        src += warps * (U * kRecord);
    };
    if (lane == 0)
        for (int i = 0; i < SLOTS; ++i)
            if (warp + i * warps < chunks) issue(warp + i * warps, i);
    __syncwarp();
    float acc[RT][NT][4];
#pragma unroll
    for (int i = 0; i < RT * NT * 4; ++i) (&acc[0][0][0])[i] = 0.f;
    // A lane without a token reads the last one's: a product's columns do not
    // mix, and its column is not stored.
    const __half* xrow[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) xrow[nt] = p.x + (int64_t)min(t0 + 8 * nt + g, p.n - 1) * p.s.in + 8 * t4;

    int slot = 0;
    uint32_t parity = 0;
    for (int c = warp; c < chunks; c += warps) {
        // the copy that never comes is recorded; the later ones land first (bounded)
        if (!__all_sync(0xffffffffu, mbar_wait(&full[slot], parity))) {
            if (lane == 0) {
                record_status(p.status, HX_ERR_TIMEOUT);
                for (int i = 1; i < SLOTS; ++i)
                    if (c + i * warps < chunks)
                        mbar_wait(&full[(slot + i) % SLOTS], slot + i < SLOTS ? parity : parity ^ 1);
            }
            break;
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int k0 = (c * U + j) * kW4Unit;
            if (U > 1 && k0 >= p.s.in) break;
            uint4 x[4][NT];
            if (k0 + kW4Unit <= p.s.in) {
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) x[q][nt] = *reinterpret_cast<const uint4*>(xrow[nt] + k0 + 32 * q);
            } else {  // the last unit of inputs that are no multiple of 128
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        x[q][nt] = k0 + 32 * q < p.s.in ? *reinterpret_cast<const uint4*>(xrow[nt] + k0 + 32 * q)
                                                        : make_uint4(0, 0, 0, 0);
            }
            const uint8_t* rec = ring + slot * kSlot + j * kRecord;
#pragma unroll
            for (int r = 0; r < RT; ++r, rec += U * kRecord) {
                float dot[NT][4];
                uint4 w;
#pragma unroll
                for (int q = 0; q < 4; ++q) {  // 32 inputs each: block q / 2, steps 2 (q % 2) and + 1
                    if (q % 2 == 0) w = *reinterpret_cast<const uint4*>(rec + (q / 2) * 512 + 16 * lane);
                    // 1024 + z for the low row (lane's row g), 64 + z for the high one (g + 8)
                    uint32_t lo_off = 0x64086408u, hi_off = 0x54805480u;
                    if constexpr (ZEROS) {
                        const uint32_t z = *reinterpret_cast<const uint16_t*>(rec + kCodes + kScales +
                                                                              (q / kPer) * kW4Rows + 2 * g);
                        lo_off = (0x6400u + (z & 0xff)) * 0x10001u;     // one unit of z is one bit
                        hi_off = (0x5400u + (z >> 8 << 4)) * 0x10001u;  // or sixteen
                    }
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        const uint32_t wd = q % 2 ? (s ? w.w : w.z) : (s ? w.y : w.x), we = wd >> 8;
                        uint32_t a[4];
                        a[0] = h2_sub(lop_and_or(wd, 0x000f000fu, 0x64006400u), lo_off);
                        a[1] = h2_sub(lop_and_or(wd, 0x00f000f0u, 0x54005400u), hi_off);
                        a[2] = h2_sub(lop_and_or(we, 0x000f000fu, 0x64006400u), lo_off);
                        a[3] = h2_sub(lop_and_or(we, 0x00f000f0u, 0x54005400u), hi_off);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const uint4& xv = x[q][nt];
                            const uint32_t b0 = s ? xv.z : xv.x, b1 = s ? xv.w : xv.y;
                            if (q % kPer == 0 && s == 0) mma_16816_first(dot[nt], a, b0, b1);
                            else mma_16816(dot[nt], a, b0, b1);
                        }
                    }
                    if (q % kPer == kPer - 1) {
                        const float2 sf = __half22float2(*reinterpret_cast<const __half2*>(
                            rec + kCodes + (q / kPer) * kW4Rows * 2 + 4 * g));
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            acc[r][nt][0] = fmaf(sf.x, dot[nt][0], acc[r][nt][0]);
                            acc[r][nt][1] = fmaf(sf.x, dot[nt][1], acc[r][nt][1]);
                            acc[r][nt][2] = fmaf(sf.y, dot[nt][2], acc[r][nt][2]);
                            acc[r][nt][3] = fmaf(sf.y, dot[nt][3], acc[r][nt][3]);
                        }
                    }
                }
            }
        }
        __syncwarp();  // the slot has been read
        if (lane == 0 && c + SLOTS * warps < chunks) issue(c + SLOTS * warps, slot);
        if (++slot == SLOTS) {
            slot = 0;
            parity ^= 1;
        }
    }
    // Every copy has landed (a warp waits for all of its own), every lane has
    // read its last slot: the ring's place is free for the partial sums.
    __syncwarp();
    float* mine = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                mine[(16 * r + g + 8 * (e >> 1)) * kCols + 8 * nt + 2 * t4 + (e & 1)] = acc[r][nt][e];
    __syncthreads();
    for (int i = threadIdx.x; i < RT * 16 * 8 * NT; i += blockDim.x) {
        const int r = i % (RT * 16), t = t0 + i / (RT * 16);
        const int64_t row = tile0 * 16 + r;
        if (t >= p.n || row >= p.s.out) continue;
        float y = 0.f;
        for (int w = 0; w < warps; ++w)
            y += reinterpret_cast<const float*>(smem + (size_t)w * SLOTS * kSlot)[r * kCols + i / (RT * 16)];
        if (p.bias) y += __half2float(p.bias[row]);
        const int64_t at = (int64_t)t * p.s.out + row;
        if (p.y_f32) static_cast<float*>(p.y)[at] = y;
        else static_cast<__half*>(p.y)[at] = __float2half_rn(y);
    }
}

template <int NT, int RT, int U, int SLOTS, int GROUP, bool ZEROS>
static int launch_w4(const W4Params& p, int warps, cudaStream_t stream)
{
    auto kernel = w4_linear_kernel<NT, RT, U, SLOTS, GROUP, ZEROS>;
    const dim3 grid((p.s.tiles + RT - 1) / RT, (p.n + 8 * NT - 1) / (8 * NT));
    const int smem = warps * SLOTS * RT * U * p.s.record;
    static std::atomic<bool> attr_set[64];  // per device; set again on ordinals past 63
    int dev = 0;
    HX_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !attr_set[dev].load(std::memory_order_acquire)) {
        HX_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
        if (dev >= 0 && dev < 64) attr_set[dev].store(true, std::memory_order_release);
    }
    kernel<<<grid, warps * 32, smem, stream>>>(p);
    return check_launch("w4_linear_kernel");
}

template <int NT, int RT, int U, int SLOTS>
static int launch_w4_group(const W4Params& p, int warps, bool zeros, cudaStream_t s)
{
    if (p.s.group == 32) return zeros ? launch_w4<NT, RT, U, SLOTS, 32, true>(p, warps, s)
                                      : launch_w4<NT, RT, U, SLOTS, 32, false>(p, warps, s);
    if (p.s.group == 64) return zeros ? launch_w4<NT, RT, U, SLOTS, 64, true>(p, warps, s)
                                      : launch_w4<NT, RT, U, SLOTS, 64, false>(p, warps, s);
    return zeros ? launch_w4<NT, RT, U, SLOTS, 128, true>(p, warps, s)
                 : launch_w4<NT, RT, U, SLOTS, 128, false>(p, warps, s);
}

// Row tiles that share x: enough that x is no more data than the weights; warps to fill the GPU.
template <int NT>
static int launch_w4_shape(const W4Params& p, bool zeros, cudaStream_t stream)
{
    const int sms = num_sms();
    int rt = std::min(4, (p.n + 1) / 2);
    rt = rt >= 4 ? 4 : rt >= 2 ? 2 : 1;
    if (NT == 4) rt = 2;
    while (rt > (NT == 1 ? 1 : 2) && p.s.tiles < rt * sms) rt /= 2;
    const int ctas = (p.s.tiles + rt - 1) / rt;
    int warps = 4;
    while (warps < kW4MaxWarps && ctas * warps * 2 <= sms * 24 && warps * 2 <= p.s.units) warps *= 2;
    if constexpr (NT == 1)
        if (rt == 1) return launch_w4_group<NT, 1, 2, 3>(p, warps, zeros, stream);
    if constexpr (NT <= 2)
        if (rt == 4) return launch_w4_group<NT, 4, 1, 2>(p, warps, zeros, stream);
    return launch_w4_group<NT, 2, 1, 3>(p, warps, zeros, stream);
}

static int check_w4(int out, int in, int group, bool zeros, W4Shape& s)
{
    if (!w4_shape(out, in, group, zeros, s))
        return fail(HX_ERR_INVALID, "weight [%d][%d] with groups of %d: groups are 32, 64 or 128 and divide the "
                    "inputs", out, in, group);
    return HX_OK;
}

static bool misaligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }

}  // namespace hx

using namespace hx;

extern "C" size_t hx_w4_packed_bytes(int out_features, int in_features, int group, int with_zeros)
{
    W4Shape s;
    return w4_shape(out_features, in_features, group, with_zeros != 0, s) ? s.bytes : 0;
}

extern "C" int hx_w4_pack(const uint8_t* codes, const void* scales, const uint8_t* zeros,
                          int out_features, int in_features, int group, void* packed,
                          size_t packed_bytes, hx_stream_t stream)
{
    HX_NVTX_RANGE("hx_w4_pack");
    W4Shape s;
    if (int rc = check_w4(out_features, in_features, group, zeros != nullptr, s)) return rc;
    if (!codes || !scales || !packed) return fail(HX_ERR_INVALID, "null codes/scales/packed");
    if (misaligned(scales, 2) || misaligned(packed, 16))
        return fail(HX_ERR_INVALID, "scales must be 2-byte and the packed weight 16-byte aligned");
    if (packed_bytes < s.bytes)
        return fail(HX_ERR_INVALID, "packed weight of %zu bytes < %zu needed", packed_bytes, s.bytes);
    const int blocks = (int)std::min<int64_t>((int64_t)s.tiles * s.units, (int64_t)num_sms() * 64);
    w4_pack_kernel<<<blocks, 256, 0, (cudaStream_t)stream>>>(codes, (const __half*)scales, zeros, s, (char*)packed);
    return check_launch("w4_pack_kernel");
}

extern "C" int hx_w4_quantize(const void* w, int out_features, int in_features, int group,
                              uint8_t* codes, void* scales, hx_stream_t stream)
{
    HX_NVTX_RANGE("hx_w4_quantize");
    W4Shape s;
    if (int rc = check_w4(out_features, in_features, group, false, s)) return rc;
    if (!w || !codes || !scales) return fail(HX_ERR_INVALID, "null w/codes/scales");
    if (misaligned(w, 2) || misaligned(scales, 2)) return fail(HX_ERR_INVALID, "w and scales must be 2-byte aligned");
    const int64_t groups = (int64_t)out_features * (in_features / group);
    const int blocks = (int)std::min<int64_t>((groups + 7) / 8, (int64_t)num_sms() * 64);
    w4_quantize_kernel<<<blocks, 256, 0, (cudaStream_t)stream>>>((const __half*)w, groups, group, codes,
                                                                 (__half*)scales);
    return check_launch("w4_quantize_kernel");
}

extern "C" int hx_w4_linear(const void* x, int n_tokens, int in_features, const void* packed,
                            size_t packed_bytes, int out_features, int group, int with_zeros,
                            const void* bias, void* y, int y_dtype, hx_stream_t stream)
{
    HX_NVTX_RANGE("hx_w4_linear");
    W4Params p{};
    if (int rc = check_w4(out_features, in_features, group, with_zeros != 0, p.s)) return rc;
    if (n_tokens < 0 || n_tokens > 65535 * 32)
        return fail(HX_ERR_INVALID, "n_tokens %d outside [0, %d]", n_tokens, 65535 * 32);
    if (y_dtype != HX_FP16 && y_dtype != HX_FP32) return fail(HX_ERR_INVALID, "y dtype %d", y_dtype);
    if (n_tokens == 0) return HX_OK;
    if (!x || !packed || !y) return fail(HX_ERR_INVALID, "null x/packed/y");
    if (misaligned(x, 16) || misaligned(packed, 16))
        return fail(HX_ERR_INVALID, "x and the packed weight must be 16-byte aligned");
    if (misaligned(y, y_dtype == HX_FP32 ? 4 : 2) || misaligned(bias, 2))
        return fail(HX_ERR_INVALID, "y and bias must be aligned to their elements");
    if (packed_bytes < p.s.bytes)
        return fail(HX_ERR_INVALID, "packed weight of %zu bytes < %zu needed", packed_bytes, p.s.bytes);
    p.x = (const __half*)x;
    p.packed = (const char*)packed;
    p.bias = (const __half*)bias;
    p.y = y;
    p.n = n_tokens;
    p.y_f32 = y_dtype == HX_FP32;
    p.status = status_word();
    cudaStream_t s = (cudaStream_t)stream;
    if (n_tokens <= 8) return launch_w4_shape<1>(p, with_zeros != 0, s);
    if (n_tokens <= 16) return launch_w4_shape<2>(p, with_zeros != 0, s);
    return launch_w4_shape<4>(p, with_zeros != 0, s);
}
