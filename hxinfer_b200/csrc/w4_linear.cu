// w4_linear.cu — projections of a few tokens with 4-bit weights: quantisation,
// layout and the product y = W x + b.  Beside hx_qkv_rope_append (fp16
// weights): a decode step reads every weight once, so a quarter of the bytes
// is up to a quarter of the time.  The reference engine has no counterpart
// (its linear layers are cuBLAS GEMVs over fp16/fp32, matmul_cuda.cu:106-189).
//
//   y[t][o] = sum_g s[o][g] * ( sum_{k in g} (c[o][k] - z[o][g]) x[t][k] ) + b[o]
//
// The bound is HBM (the weights): 6.5 TB/s are 45 weights a cycle and SM.  An fp16
// mma.sync (16 rows by 8 tokens by 16 inputs) takes one of the SM's four tensor
// pipes 8 cycles, the SM 2.0 (measured in a loop without loads, the same for the
// integer one of twice the inputs): 128 weights a cycle for up to 8 tokens, 32
// for 32.  What the weights cost on the way there, conversion and sums, differs
// with the number of tokens; hence a kernel for each range of them.
//
// 1-2 tokens, w4_vector_kernel: integers.  x becomes fixed point, 31 bits with a
// power of two per group (exact from 2^-18 of the group's largest |x| on, off by
// at most 2^-30 of it below: a 64th of an fp32 rounding of a sum that it is part
// of), as four signed digits of base 256 per token: columns of the B operand of
// mma.sync m16n8k32 (u8 by s8, 32-bit sums, exact).  The codes are the A operand
// as they stand, one mask for four of them, 256 a cycle and SM.  Scales, zero
// points and the digits' weights are applied to a group's sums in fp32.  Every
// CTA puts all of x into fixed point, some 0.05 us per 128 inputs and token.  It is
// taken wherever that fits (launch_w4_vector_group gives the limit and what it
// takes against the next kernel).
//
// 3-32 tokens, w4_linear_kernel: c - z is a small integer, exact in fp16, so a
// group's sum is a product of fp16 values on the tensor cores with fp32
// accumulation, and its scale is applied in fp32: nothing is rounded before y.
// No unit is near its limit (8 x 8192 x 28672, 36.6 us: tensor pipes 15 % busy,
// issue slots 34 %, DRAM 2.8 TB/s under the profiler): the grid is 896 CTAs of
// which 740 fit at once, so a second round runs on a fifth of the GPU, and a
// warp's copies, conversion and products follow each other.
//
// More tokens: w4_tile.cu, the same sums on tcgen05.  (For few tokens a tcgen05
// product of 128 rows by 16 inputs costs some 100 cycles whatever the number of
// tokens, and its operand has to be converted into tensor or shared memory
// first: 8 x 8192 x 28672 took 67 us that way, 36.6 here.)
//
// Layout of a packed weight (rows padded to 16, inputs to 128): for every tile
// of 16 rows, for every unit of 128 inputs, one record of
//   codes  [2 blocks of 64 inputs][32 lanes][4 words]
//   scales [groups][8][2] fp16, rows g and g + 8 of the tile in a pair
//   zeros  [groups][8][2] bytes, likewise (only with zero points)
// so that a warp's share of a row tile is one stream of memory, fetched by
// bulk copies into a ring of the warp's own.
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

#include "hx_w4.cuh"

namespace hx {

constexpr int kW4MaxWarps = 16;
constexpr int kW4VectorSlots = 2;  // 1-2 tokens: copies in flight per warp
constexpr int kW4VectorSmem = 224 * 1024;

// More tokens' sums and x need more registers than 16 warps on an SM leave.
constexpr int w4_max_warps(int nt, int group) { return nt <= 2 ? kW4MaxWarps : group >= (nt == 3 ? 64 : 128) ? 12 : 8; }

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

// D = A(16x16 fp16, row) * B(16x8 fp16, col): the first product of a sum.
__device__ __forceinline__ void mma_16816_first(float* d, const uint32_t* a, uint32_t b0, uint32_t b1)
{
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// One CTA per (RT row tiles, token group of 8 NT).  Its warps take 128-input
// units in turn, U at a time, for all RT tiles, and add their partial sums in
// shared memory in a fixed order.  RT tiles share the x operand, which for
// several tokens is more data than one tile's weights.
template <int NT, int RT, int U, int SLOTS, int GROUP, bool ZEROS>
__global__ void __launch_bounds__(w4_max_warps(NT, GROUP) * 32, 1) w4_linear_kernel(const W4Params p)
{
    constexpr int kGroups = kW4Unit / GROUP;  // groups in a unit
    constexpr int kPer = GROUP / 32;          // 32-input quarters in a group
    constexpr int kCodes = kW4Rows * kW4Unit / 2, kScales = kGroups * kW4Rows * 2;
    constexpr int kRecord = kCodes + kScales + (ZEROS ? kGroups * kW4Rows : 0);
    constexpr int kSlot = RT * U * kRecord;   // bytes
    constexpr int kCols = 8 * NT + 1;         // a warp's partial sums [16 RT][8 NT + 1] take its ring's place
    static_assert(SLOTS * kSlot >= RT * 16 * kCols * 4, "partial sums");
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ uint64_t bars[w4_max_warps(NT, GROUP)][SLOTS];
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
    pdl_wait();  // x, and perhaps the weight, come from earlier kernels on the stream
    pdl_trigger();  // not before: a dependent may read early what kernels before this one wrote
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
    cudaError_t e = launch_kernel(kernel, grid, dim3(warps * 32), smem, stream, true, p);
    if (e != cudaSuccess) return cuda_fail(e, "w4_linear_kernel launch");
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

// Two row tiles share the x operand, which comes from L2 once per CTA (8 tokens
// x 8192 x 28672: 34.1 us, 38.9 with four); one where two would leave SMs idle.
// Warps: as many as keep an SM's registers in use.  Three and four n-tiles need
// more than 128 registers, so 12 warps of them fill an SM, in one CTA, two or
// three.
template <int NT>
static int launch_w4_shape(const W4Params& p, bool zeros, cudaStream_t stream)
{
    const int sms = num_sms();
    const int rt = NT == 1 && p.s.tiles < 2 * sms ? 1 : 2;
    const int ctas = (p.s.tiles + rt - 1) / rt;
    const int most = w4_max_warps(NT, p.s.group);
    int warps = 4;
    if (NT > 2) warps = std::min(std::max(most / ((ctas + sms - 1) / sms), 4), std::max(p.s.units, 4));
    else while (warps < most && ctas * warps * 2 <= sms * 24 && warps * 2 <= p.s.units) warps *= 2;
    if constexpr (NT == 1)
        if (rt == 1) return launch_w4_group<NT, 1, 2, 3>(p, warps, zeros, stream);
    return launch_w4_group<NT, 2, 1, 3>(p, warps, zeros, stream);
}

// ------------------------------------------------------------------ 1-2 tokens

constexpr int kW4Digits = 4;  // of x in fixed point

// Columns of x's digits, and units of a copy (two tokens' digits and sums leave
// less room for the rings).
template <int TOK>
struct W4Columns {
    static constexpr int kCols = kW4Digits * TOK, kUnits = TOK == 1 ? 4 : 2;
};

// x in fixed point for one unit: COLS columns, a token's digits from the highest
// down.  Quarter q, column c: 32 bytes, t4's eight at 8 t4: inputs 8 t4 +
// {0, 2, 1, 3}, then 8 t4 + 4 + {0, 2, 1, 3}, the order of a word's nibbles.  Per
// group: the columns' sums and factors.
template <int COLS>
struct W4Fixed {
    uint32_t bytes[4][COLS][8];
    int sums[4][COLS];
    float factor[4][COLS];
};

// Fills fx[0], fx[step], ... below fx[count] with the units u0, u0 + step, ...,
// by one warp; lane l holds inputs 4 l .. 4 l + 3 of a unit.
template <int TOK, int COLS, int GROUP>
__device__ void w4_fix_x(const W4Params& p, W4Fixed<COLS>* fx, int u0, int count, int step, int lane)
{
    constexpr int kAhead = 4;  // loads in flight
    uint2 next[kAhead];
    count = (count + step - 1) / step;  // units of this warp
    auto load = [&](int i) {
        const int k = (u0 + i / TOK * step) * kW4Unit + 4 * lane;
        return i < count * TOK && k < p.s.in
            ? *reinterpret_cast<const uint2*>(p.x + (int64_t)(i % TOK) * p.s.in + k) : make_uint2(0, 0);
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) next[i] = load(i);
    for (int i = 0; i < count * TOK; ++i) {
        const int t = i % TOK, unit = i / TOK * step;
        const uint2 raw = next[0];
#pragma unroll
        for (int e = 0; e + 1 < kAhead; ++e) next[e] = next[e + 1];
        next[kAhead - 1] = load(i + kAhead);
        float v[4];
        {
            const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&raw.x));
            const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&raw.y));
            v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
        }
        // the largest |x| of the group, as bits (NaN sorts above infinity)
        uint32_t mx = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = max(mx, __float_as_uint(fabsf(v[e])));
#pragma unroll
        for (int o = GROUP / 8; o; o >>= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const int exp = (int)(mx >> 23);  // biased; 255: an infinity or NaN, 0: all zero (fp16's least is 2^-24)
        const bool plain = exp != 0 && exp != 255;
        const float scale = __uint_as_float((uint32_t)(127 + 29 + 127 - exp) << 23);  // 2^29 / 2^floor(log2 max)
        uint32_t digit[kW4Digits] = {0, 0, 0, 0};
        int sums[kW4Digits] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            // |f| < 2^30 in signed digits of base 256: the high one stays below 66
            const int f = plain ? __float2int_rn(v[e] * scale) : 0;
            const int d0 = (int)(int8_t)f, f1 = (f - d0) >> 8, d1 = (int)(int8_t)f1, f2 = (f1 - d1) >> 8;
            const int d2 = (int)(int8_t)f2, d3 = (f2 - d2) >> 8;
            const int d[kW4Digits] = {d3, d2, d1, d0};
            constexpr int kByte[4] = {0, 2, 1, 3};  // input e's byte in its word
#pragma unroll
            for (int q = 0; q < kW4Digits; ++q) {
                digit[q] |= (uint32_t)(d[q] & 255) << (8 * kByte[e]);
                sums[q] += d[q];
            }
        }
#pragma unroll
        for (int q = 0; q < kW4Digits; ++q) {
#pragma unroll
            for (int o = GROUP / 8; o; o >>= 1) sums[q] += __shfl_xor_sync(0xffffffffu, sums[q], o);
            fx[unit].bytes[lane >> 3][kW4Digits * t + q][lane & 7] = digit[q];
            if (4 * lane % GROUP == 0) {
                fx[unit].sums[4 * lane / GROUP][kW4Digits * t + q] = sums[q];
                const float one = exp == 255 ? __uint_as_float(0x7fffffffu) : exp == 0 ? 0.f
                                                   : __uint_as_float((uint32_t)(exp - 29) << 23);
                fx[unit].factor[4 * lane / GROUP][kW4Digits * t + q] = one * (float)(1 << 8 * (kW4Digits - 1 - q));
            }
        }
    }
}

// D = A(16x32 u8, row) * B(32x8 s8, col) + C
__device__ __forceinline__ void imma_16832(int* d, const uint32_t* a, uint32_t b0, uint32_t b1)
{
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The first product of a sum.
__device__ __forceinline__ void imma_16832_first(int* d, const uint32_t* a, uint32_t b0, uint32_t b1)
{
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%10, %10, %10, %10};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));
}

// One CTA per SM (fewer for few tiles) takes a run of row tiles; its warps
// share a tile's units, each the same slice of all its tiles, so that x is
// put into fixed point once, no warp waits for another before the end, and the
// work differs between SMs by a tile of 16 rows at most.  A warp's sums of a
// tile wait in shared memory until all are there.
template <int TOK, int GROUP, bool ZEROS>
__global__ void __launch_bounds__(kW4MaxWarps * 32, 1) w4_vector_kernel(const W4Params p, int max_tiles, int abreast)
{
    constexpr int COLS = W4Columns<TOK>::kCols, U = W4Columns<TOK>::kUnits, SLOTS = kW4VectorSlots;
    constexpr int kGroups = kW4Unit / GROUP, kPer = GROUP / 32;
    constexpr int kCodes = kW4Rows * kW4Unit / 2, kScales = kGroups * kW4Rows * 2;
    constexpr int kRecord = kCodes + kScales + (ZEROS ? kGroups * kW4Rows : 0), kSlot = U * kRecord;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ uint64_t bars[kW4MaxWarps][SLOTS];
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    // tiles [tile0, tile0 + tiles) of the CTA, `abreast` at a time; units
    // [u0, u0 + count) of the warp, in chunks of U
    const int tile0 = (int)((int64_t)p.s.tiles * blockIdx.x / gridDim.x);
    const int tiles = (int)((int64_t)p.s.tiles * (blockIdx.x + 1) / gridDim.x) - tile0;
    const int ways = warps / abreast, way = warp % ways, first = warp / ways;
    const int u0 = p.s.units * way / ways, count = p.s.units * (way + 1) / ways - u0;
    const int chunks = (count + U - 1) / U * ((tiles - first + abreast - 1) / abreast);
    uint8_t* ring = smem + (size_t)warp * SLOTS * kSlot;
    float* part = reinterpret_cast<float*>(smem + (size_t)warps * SLOTS * kSlot);  // [max_tiles][ways][16][COLS]
    auto* fx = reinterpret_cast<W4Fixed<COLS>*>(part + (size_t)max_tiles * ways * kW4Rows * COLS);
    uint64_t* full = bars[warp];
    const uint64_t pol = l2_evict_first_policy();
    const char* src = p.packed + ((int64_t)(tile0 + first) * p.s.units + u0) * kRecord;  // of the next chunk to copy
    const int64_t skip = ((int64_t)abreast * p.s.units - count) * kRecord;
    int ahead = 0;  // units of the tile copied before it
    auto issue = [&](int slot) {  // lane 0
        const int n = min(U, count - ahead);
        mbar_arrive_expect_tx(&full[slot], n * kRecord);
        bulk_load(ring + slot * kSlot, src, n * kRecord, &full[slot], pol);
        src += n * kRecord;
        ahead += n;
        if (ahead == count) {
            ahead = 0;
            src += skip;
        }
    };
    if (lane == 0) {
        for (int i = 0; i < SLOTS; ++i) mbar_init(&full[i], 1);
        fence_mbar_init();
    }
    pdl_wait();  // x, and perhaps the weight, come from earlier kernels on the stream
    pdl_trigger();  // not before: a dependent may read early what kernels before this one wrote
    if (lane == 0)
        for (int i = 0; i < SLOTS && i < chunks; ++i) issue(i);
    // the `abreast` warps that take the same units convert every other one each
    w4_fix_x<TOK, COLS, GROUP>(p, fx + u0 + first, u0 + first, count - first, abreast, lane);
    __syncwarp();
    if (abreast > 1) asm volatile("bar.sync %0, %1;" ::"r"(1 + way), "r"(32 * abreast) : "memory");  // at most 8 ways
    int slot = 0;
    uint32_t parity = 0;
    for (int c = 0, tile = first; tile < tiles; tile += abreast) {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};  // rows g, g + 8 x columns 2 t4, 2 t4 + 1
        const W4Fixed<COLS>* f = fx + u0;
        for (int left = count; left > 0; left -= U, ++c) {
            // the copy that never comes is recorded; the later ones land first (bounded)
            if (!__all_sync(0xffffffffu, mbar_wait(&full[slot], parity))) {
                if (lane == 0) {
                    record_status(p.status, HX_ERR_TIMEOUT);
                    for (int i = 1; i < SLOTS && c + i < chunks; ++i)
                        mbar_wait(&full[(slot + i) % SLOTS], slot + i < SLOTS ? parity : parity ^ 1);
                }
                tile = tiles;
                break;
            }
            const uint8_t* rec = ring + slot * kSlot;
#pragma unroll
            for (int j = 0; j < U; ++j, rec += kRecord, ++f) {
                if (j > 0 && j >= left) break;
                uint4 w[2];
#pragma unroll
                for (int b = 0; b < 2; ++b) w[b] = *reinterpret_cast<const uint4*>(rec + b * 512 + 16 * lane);
                int d[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {  // 32 inputs each
                    const uint4& wb = w[q / 2];
                    const uint32_t w0 = q % 2 ? wb.z : wb.x, w1 = q % 2 ? wb.w : wb.y;
                    // even nibbles are row g's; odd ones, sixteen times their code
                    // where they stand, row g + 8's
                    const uint32_t a[4] = {w0 & 0x0f0f0f0fu, w0 & 0xf0f0f0f0u, w1 & 0x0f0f0f0fu, w1 & 0xf0f0f0f0u};
                    const uint2 x = *reinterpret_cast<const uint2*>(&f->bytes[q][g % COLS][2 * t4]);
                    if (q % kPer == 0) imma_16832_first(d, a, x.x, x.y);
                    else imma_16832(d, a, x.x, x.y);
                    if (q % kPer == kPer - 1) {
                        const int grp = q / kPer;
                        const float2 sf = __half22float2(*reinterpret_cast<const __half2*>(rec + kCodes + grp * kW4Rows * 2 + 4 * g));
                        int z0 = 8, z1 = 8;
                        if constexpr (ZEROS) {
                            const uint32_t z = *reinterpret_cast<const uint16_t*>(rec + kCodes + kScales + grp * kW4Rows + 2 * g);
                            z0 = z & 0xff;
                            z1 = z >> 8;
                        }
                        const int2 sum = *reinterpret_cast<const int2*>(&f->sums[grp][2 * t4 % COLS]);
                        const float2 fac = *reinterpret_cast<const float2*>(&f->factor[grp][2 * t4 % COLS]);
                        acc[0] = fmaf(sf.x * fac.x, (float)(d[0] - z0 * sum.x), acc[0]);
                        acc[1] = fmaf(sf.x * fac.y, (float)(d[1] - z0 * sum.y), acc[1]);
                        const float sy = sf.y * 0.0625f;
                        acc[2] = fmaf(sy * fac.x, (float)(d[2] - 16 * z1 * sum.x), acc[2]);
                        acc[3] = fmaf(sy * fac.y, (float)(d[3] - 16 * z1 * sum.y), acc[3]);
                    }
                }
            }
            __syncwarp();  // the slot has been read
            if (lane == 0 && c + SLOTS < chunks) issue(slot);
            if (++slot == SLOTS) {
                slot = 0;
                parity ^= 1;
            }
        }
        if (tile < tiles && 2 * t4 < COLS) {
            float* mine = part + ((size_t)tile * ways + way) * kW4Rows * COLS + 2 * t4;
            *reinterpret_cast<float2*>(mine + g * COLS) = make_float2(acc[0], acc[1]);
            *reinterpret_cast<float2*>(mine + (g + 8) * COLS) = make_float2(acc[2], acc[3]);
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < tiles * kW4Rows * TOK; i += blockDim.x) {
        const int r = i % (tiles * kW4Rows), t = i / (tiles * kW4Rows);
        const int64_t row = (int64_t)tile0 * kW4Rows + r;
        if (row >= p.s.out) continue;
        const float* v = part + ((size_t)(r / kW4Rows) * ways * kW4Rows + r % kW4Rows) * COLS + kW4Digits * t;
        float digit[kW4Digits] = {0.f, 0.f, 0.f, 0.f};  // digit by digit, warps in order
        for (int w = 0; w < ways; ++w, v += kW4Rows * COLS)
#pragma unroll
            for (int q = 0; q < kW4Digits; ++q) digit[q] += v[q];
        float y = (digit[0] + digit[1]) + (digit[2] + digit[3]);
        if (p.bias) y += __half2float(p.bias[row]);
        const int64_t at = (int64_t)t * p.s.out + row;
        if (p.y_f32) static_cast<float*>(p.y)[at] = y;
        else static_cast<__half*>(p.y)[at] = __float2half_rn(y);
    }
}


template <int TOK, int GROUP, bool ZEROS>
static int launch_w4_vector(const W4Params& p, int ctas, int warps, int abreast, int smem, cudaStream_t stream)
{
    auto kernel = w4_vector_kernel<TOK, GROUP, ZEROS>;
    static std::atomic<bool> attr_set[64];  // per device; set again on ordinals past 63
    int dev = 0;
    HX_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !attr_set[dev].load(std::memory_order_acquire)) {
        HX_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kW4VectorSmem));
        if (dev >= 0 && dev < 64) attr_set[dev].store(true, std::memory_order_release);
    }
    cudaError_t e = launch_kernel(kernel, dim3(ctas), dim3(warps * 32), smem, stream, true, p,
                                  (p.s.tiles + ctas - 1) / ctas, abreast);
    if (e != cudaSuccess) return cuda_fail(e, "w4_vector_kernel launch");
    return check_launch("w4_vector_kernel");
}

// The kernel for 1-2 tokens, or HX_ERR_UNSUPPORTED (nothing launched, no
// message) when x in fixed point and the sums do not fit beside the rings: past
// 17,920 inputs with one token and groups of 128, 13,824 with groups of 32 and
// zero points, 15,360 and 14,336 with two.  The call then takes w4_linear_kernel.
// In a graph, this kernel / that one, us: 1 x 4096 x 14336 8.4 / 14.5, 1 x 8192 x
// 8192 10.8 / 14.2, 1 x 8192 x 28672 23.5 / 31.3, 1 x 14336 x 4096 12.1 / 11.9,
// 2 x 4096 x 14336 11.3 / 14.4.  It loses where a CTA has one or two row tiles to
// set its conversion of x against: 1 x 4096 x 1024 4.0 / 2.9, 2 x 4096 x 4096
// 7.3 / 5.1, 1 x 17920 x 4096 25.3 / 14.5 (the sums of one tile fit, so two rounds).
template <int TOK>
static int launch_w4_vector_group(const W4Params& p, bool zeros, cudaStream_t s)
{
    using Columns = W4Columns<TOK>;
    const int sms = num_sms();
    // a warp's slice of a tile should be a few units long: with few units, and
    // tiles enough, two tiles at a time (1 x 3584 x 37888: 18.5 us, 19.8 with one
    // or four; 2 x 4096 x 14336: 13.0, 15.0 with one)
    const int abreast = p.s.units < 4 * kW4MaxWarps && p.s.tiles >= 6 * sms ? 2 : 1;
    const int ways = std::min(kW4MaxWarps / abreast, p.s.units), warps = ways * abreast;
    // a CTA per SM, or several rounds of them where the sums of so many tiles
    // would not fit beside the rings and x
    const size_t fixed = (size_t)warps * kW4VectorSlots * Columns::kUnits * p.s.record +
                         p.s.units * sizeof(W4Fixed<Columns::kCols>);
    const size_t per_tile = (size_t)ways * kW4Rows * Columns::kCols * sizeof(float);
    if (fixed + per_tile > (size_t)kW4VectorSmem) return HX_ERR_UNSUPPORTED;
    const int fit = (int)std::min<size_t>(((size_t)kW4VectorSmem - fixed) / per_tile, 1 << 16);
    const int64_t rounds = (p.s.tiles + (int64_t)sms * fit - 1) / ((int64_t)sms * fit);
    const int ctas = (int)std::min<int64_t>(p.s.tiles, rounds * sms);
    const size_t smem = fixed + (size_t)((p.s.tiles + ctas - 1) / ctas) * per_tile;
    const int b = (int)smem;
    if (p.s.group == 32) return zeros ? launch_w4_vector<TOK, 32, true>(p, ctas, warps, abreast, b, s)
                                      : launch_w4_vector<TOK, 32, false>(p, ctas, warps, abreast, b, s);
    if (p.s.group == 64) return zeros ? launch_w4_vector<TOK, 64, true>(p, ctas, warps, abreast, b, s)
                                      : launch_w4_vector<TOK, 64, false>(p, ctas, warps, abreast, b, s);
    return zeros ? launch_w4_vector<TOK, 128, true>(p, ctas, warps, abreast, b, s)
                 : launch_w4_vector<TOK, 128, false>(p, ctas, warps, abreast, b, s);
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
    status_word();  // allocated here, so that the first hx_w4_linear may be captured into a graph
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
    // CTAs store while others still read all of x
    const uintptr_t x0 = reinterpret_cast<uintptr_t>(x), y0 = reinterpret_cast<uintptr_t>(y);
    const uint64_t x_bytes = (uint64_t)n_tokens * in_features * 2;
    const uint64_t y_bytes = (uint64_t)n_tokens * out_features * (y_dtype == HX_FP32 ? 4 : 2);
    if (x0 < y0 + y_bytes && y0 < x0 + x_bytes) return fail(HX_ERR_INVALID, "y overlaps x");
    p.x = (const __half*)x;
    p.packed = (const char*)packed;
    p.bias = (const __half*)bias;
    p.y = y;
    p.n = n_tokens;
    p.y_f32 = y_dtype == HX_FP32;
    p.status = status_word();
    cudaStream_t s = (cudaStream_t)stream;
    if (n_tokens <= 2) {
        const int rc = n_tokens == 1 ? launch_w4_vector_group<1>(p, with_zeros != 0, s)
                                     : launch_w4_vector_group<2>(p, with_zeros != 0, s);
        if (rc != HX_ERR_UNSUPPORTED) return rc;
    }
    if (n_tokens > 32) return launch_w4_tile(p, with_zeros != 0, s);
    if (n_tokens <= 8) return launch_w4_shape<1>(p, with_zeros != 0, s);
    if (n_tokens <= 16) return launch_w4_shape<2>(p, with_zeros != 0, s);
    if (n_tokens <= 24) return launch_w4_shape<3>(p, with_zeros != 0, s);
    return launch_w4_shape<4>(p, with_zeros != 0, s);
}
