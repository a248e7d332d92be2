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
// Layout of a packed weight (rows padded to 16, inputs to 128):
//   codes  [rows/16][inputs/64][32 lanes][4 words]
//   scales [rows/16][groups][8][2] fp16, rows g and g + 8 of a tile in a pair
//   zeros  [rows/16][groups][8][2] bytes, likewise (only with zero points)
// One warp-wide 16-byte load is the A operand of four m16n8k16 products, 16
// rows by 64 inputs.  Which input stands at which k of the product is free as
// long as both operands agree, so lane (g, t4) holds for k step s the inputs
//   64 b + 32 (s / 2) + 8 t4 + 4 (s % 2) + {0, 1, 2, 3}
// of rows g and g + 8: a step stays inside one group of 32, and the lane's x
// operand is two contiguous 16-byte chunks, read from global memory without
// staging.  Word s holds those eight codes as nibbles (0, 4) = row g, inputs
// 0 and 1; (1, 5) = row g + 8, inputs 0 and 1; (2, 6) and (3, 7) = inputs 2
// and 3: one mask each turns a nibble pair into two fp16 (1024 + c), or
// (1024 + 16 c) for the odd ones.
#include <algorithm>

#include "hx_common.cuh"

namespace hx {

constexpr int kW4Rows = 16;
constexpr int kW4Unit = 128;   // inputs one warp takes at a time: two 64-input blocks
constexpr int kW4Warps = 8;

struct W4Shape {
    int out, in, group;
    int tiles, units, groups;   // of the padded weight
    size_t scales_at, zeros_at, bytes;
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
    s.groups = s.units * (kW4Unit / group);
    s.scales_at = (size_t)s.tiles * s.units * kW4Unit * kW4Rows / 2;
    s.zeros_at = s.scales_at + (size_t)s.tiles * s.groups * kW4Rows * 2;
    s.bytes = s.zeros_at + (zeros ? (size_t)s.tiles * s.groups * kW4Rows : 0);
    return true;
}

// One thread per packed word, then per scale pair: gathers the codes (padding
// is 0, under a scale of 0).
__global__ void w4_pack_kernel(const uint8_t* __restrict__ codes, const __half* __restrict__ scales,
                               const uint8_t* __restrict__ zeros, W4Shape s, char* __restrict__ packed)
{
    const int64_t stride = (int64_t)gridDim.x * blockDim.x;
    const int64_t first = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t words = (int64_t)s.scales_at / 4;
    for (int64_t i = first; i < words; i += stride) {
        const int step = (int)(i & 3), lane = (int)(i >> 2) & 31, g = lane >> 2, t4 = lane & 3;
        const int64_t blk = i >> 7;  // tile * (2 units) + block
        const int64_t tile = blk / (2 * s.units);
        const int k0 = (int)(blk % (2 * s.units)) * 64 + 32 * (step / 2) + 8 * t4 + 4 * (step % 2);
        uint32_t w = 0;
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            // nibble n < 4: (row half n & 1, input 2 (n / 2)); n >= 4: the input after it
            const int64_t row = tile * kW4Rows + g + 8 * (n & 1);
            const int k = k0 + 2 * ((n & 3) >> 1) + (n >> 2);
            const uint32_t c = row < s.out && k < s.in ? codes[row * s.in + k] & 15u : 0u;
            w |= c << (4 * n);
        }
        reinterpret_cast<uint32_t*>(packed)[i] = w;
    }
    const int in_groups = s.in / s.group;
    const int64_t n_scales = (int64_t)s.tiles * s.groups * kW4Rows;
    for (int64_t i = first; i < n_scales; i += stride) {
        const int r = (int)(i & 15);
        const int64_t tile = (i >> 4) / s.groups;
        const int grp = (int)((i >> 4) % s.groups);
        const int64_t row = tile * kW4Rows + (r >> 1) + 8 * (r & 1);
        const bool in = row < s.out && grp < in_groups;
        reinterpret_cast<__half*>(packed + s.scales_at)[i] = in ? scales[row * in_groups + grp] : __float2half(0.f);
        if (zeros)
            reinterpret_cast<uint8_t*>(packed + s.zeros_at)[i] = in ? zeros[row * in_groups + grp] & 15 : 0;
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

__device__ __forceinline__ uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c)
{
    const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b),
                              *reinterpret_cast<const __half2*>(&c));
    return *reinterpret_cast<const uint32_t*>(&r);
}

struct W4Params {
    W4Shape s;
    const __half* x;
    const char* packed;
    const __half* bias;
    void* y;
    int n, y_f32;
};

// One CTA per (16-row tile, token group of 8 NT); its eight warps take the
// weight's 128-input units in turn and add their partial sums in shared
// memory in a fixed order.
template <int NT, int GROUP, bool ZEROS>
__global__ void __launch_bounds__(kW4Warps * 32) w4_linear_kernel(const W4Params p)
{
    __shared__ float part[kW4Warps][kW4Rows][8 * NT + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int64_t tile = blockIdx.x;
    const int t0 = blockIdx.y * 8 * NT;
    const uint4* codes = reinterpret_cast<const uint4*>(p.packed) + tile * p.s.units * 64 + lane;
    const uint32_t* scales = reinterpret_cast<const uint32_t*>(p.packed + p.s.scales_at) + tile * p.s.groups * 8 + g;
    const uint16_t* zeros = reinterpret_cast<const uint16_t*>(p.packed + p.s.zeros_at) + tile * p.s.groups * 8 + g;
    constexpr int kGroups = kW4Unit / GROUP;  // groups in a unit
    float acc[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[nt][e] = 0.f;

    for (int u = warp; u < p.s.units; u += kW4Warps) {
        uint4 w[2], xv[2][2][NT];
        uint32_t sc[kGroups], zp[kGroups];
#pragma unroll
        for (int b = 0; b < 2; ++b) w[b] = __ldcs(codes + (u * 2 + b) * 32);
#pragma unroll
        for (int i = 0; i < kGroups; ++i) {
            sc[i] = scales[(u * kGroups + i) * 8];
            zp[i] = ZEROS ? zeros[(u * kGroups + i) * 8] : 0u;
        }
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int k = u * kW4Unit + 64 * b + 32 * c + 8 * t4;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const int t = t0 + 8 * nt + g;
                    xv[b][c][nt] = t < p.n && k < p.s.in
                        ? *reinterpret_cast<const uint4*>(p.x + (int64_t)t * p.s.in + k) : make_uint4(0, 0, 0, 0);
                }
            }
        float dot[NT][4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {  // 32 inputs each: block q / 2, steps 2 (q % 2) and + 1
            constexpr int kPer = GROUP / 32;
            if (q % kPer == 0) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) dot[nt][e] = 0.f;
            }
            // offsets that take (1024 + c) and (1024 + 16 c) / 16 to c - z, for
            // the low row (lane's row g) and the high one (g + 8)
            uint32_t lo_off = 0x64086408u, hi_off = 0xd480d480u;  // 1024 + 8, -(64 + 8)
            if constexpr (ZEROS) {
                const uint32_t z = zp[q / kPer];
                const uint32_t z0 = z & 0xff, z1 = z >> 8;
                lo_off = (0x6400u + z0) * 0x10001u;           // 1024 + z: one unit is one bit
                hi_off = (0xd400u + (z1 << 4)) * 0x10001u;    // -(64 + z): one unit is 16 bits of 2^-4
            }
            const uint32_t ws[2] = {q % 2 ? w[q / 2].z : w[q / 2].x, q % 2 ? w[q / 2].w : w[q / 2].y};
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const uint32_t wd = ws[s], we = wd >> 8;
                uint32_t a[4];
                a[0] = h2_sub(lop_and_or(wd, 0x000f000fu, 0x64006400u), lo_off);
                a[1] = h2_fma(lop_and_or(wd, 0x00f000f0u, 0x64006400u), 0x2c002c00u, hi_off);
                a[2] = h2_sub(lop_and_or(we, 0x000f000fu, 0x64006400u), lo_off);
                a[3] = h2_fma(lop_and_or(we, 0x00f000f0u, 0x64006400u), 0x2c002c00u, hi_off);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const uint4& x = xv[q / 2][q % 2][nt];
                    mma_16816(dot[nt], a, s ? x.z : x.x, s ? x.w : x.y);
                }
            }
            if (q % kPer == kPer - 1) {
                const float2 sf = __half22float2(*reinterpret_cast<const __half2*>(&sc[q / kPer]));
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    acc[nt][0] = fmaf(sf.x, dot[nt][0], acc[nt][0]);
                    acc[nt][1] = fmaf(sf.x, dot[nt][1], acc[nt][1]);
                    acc[nt][2] = fmaf(sf.y, dot[nt][2], acc[nt][2]);
                    acc[nt][3] = fmaf(sf.y, dot[nt][3], acc[nt][3]);
                }
            }
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) part[warp][g + 8 * (e >> 1)][8 * nt + 2 * t4 + (e & 1)] = acc[nt][e];
    __syncthreads();
    for (int i = threadIdx.x; i < kW4Rows * 8 * NT; i += kW4Warps * 32) {
        const int r = i % kW4Rows, t = t0 + i / kW4Rows;
        const int64_t row = tile * kW4Rows + r;
        if (t >= p.n || row >= p.s.out) continue;
        float y = 0.f;
#pragma unroll
        for (int w = 0; w < kW4Warps; ++w) y += part[w][r][i / kW4Rows];
        if (p.bias) y += __half2float(p.bias[row]);
        const int64_t at = (int64_t)t * p.s.out + row;
        if (p.y_f32) static_cast<float*>(p.y)[at] = y;
        else static_cast<__half*>(p.y)[at] = __float2half_rn(y);
    }
}

template <int NT, int GROUP>
static int launch_w4(const W4Params& p, bool zeros, cudaStream_t stream)
{
    const dim3 grid(p.s.tiles, (p.n + 8 * NT - 1) / (8 * NT));
    if (zeros) w4_linear_kernel<NT, GROUP, true><<<grid, kW4Warps * 32, 0, stream>>>(p);
    else w4_linear_kernel<NT, GROUP, false><<<grid, kW4Warps * 32, 0, stream>>>(p);
    return check_launch("w4_linear_kernel");
}

template <int NT>
static int launch_w4_group(const W4Params& p, bool zeros, cudaStream_t stream)
{
    if (p.s.group == 32) return launch_w4<NT, 32>(p, zeros, stream);
    if (p.s.group == 64) return launch_w4<NT, 64>(p, zeros, stream);
    return launch_w4<NT, 128>(p, zeros, stream);
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
    const int64_t words = (int64_t)(s.scales_at / 4);
    const int blocks = (int)std::min<int64_t>((words + 255) / 256, (int64_t)num_sms() * 64);
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
    cudaStream_t s = (cudaStream_t)stream;
    if (n_tokens <= 8) return launch_w4_group<1>(p, with_zeros != 0, s);
    if (n_tokens <= 16) return launch_w4_group<2>(p, with_zeros != 0, s);
    return launch_w4_group<4>(p, with_zeros != 0, s);
}
