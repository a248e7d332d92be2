// norm_append.cu — RMS norm of every q and k head, NeoX RoPE and the K/V
// append in one pass: hx_rope_append for models that normalise their heads.
// The reference engine has no counterpart (its attention adds a bias instead,
// hxinfer-engine/src/layer/attention.cpp:21-35).
//
// For a head x of hd elements at position p, with weight w and table row
// (c, s)[p]:
//     y = (x r) w,  r = 1 / sqrt(mean(x^2) + eps)
//     (y[d], y[d + hd/2]) <- (y[d] c - y[d + hd/2] s, y[d + hd/2] c + y[d] s)
// v is copied.  Everything is computed in fp32 and rounded once, when it is
// stored: fp16 in the cache (its format), q_out_dtype for q.
//
// Each element is read and written once with a handful of operations, so the
// bound is HBM for prompts and the chain of dependent loads (position, block
// table, table row) for decode batches.
#include <algorithm>

#include "hx_common.cuh"

namespace hx {

constexpr int kNormThreads = 128;

// VEC elements, as 16-byte accesses where they fill them (8- and 32-byte
// groups arise for an fp16 cache row of fp32 inputs and fp32 q of fp16 ones).
template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float* f)
{
    if constexpr (VEC * sizeof(T) == 16) {
        const uint4 raw = *reinterpret_cast<const uint4*>(p);
        const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = (float)t[e];
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = (float)p[e];
    }
}

template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float* f)
{
    if constexpr (VEC == 1) {
        st(p, f[0]);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int e = 0; e < VEC; e += 4)
            *reinterpret_cast<float4*>(p + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
    } else {
        uint32_t w[VEC / 2];
#pragma unroll
        for (int e = 0; e < VEC / 2; ++e) w[e] = pack_half2(f[2 * e], f[2 * e + 1]);
        if constexpr (VEC == 8) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    }
}

struct NormParams {
    KVView view;
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;  // elements between token rows
    const void *q_weight, *k_weight;       // [hd] or null (weight 1)
    const int32_t *seq_ids, *positions;
    const float2* table;                   // [table_max_pos][hd/2], or null: no rotation
    void* q_out;
    int table_max_pos, hq, rounds;
    float eps;
    int* status;
};

// grid (token, slot chunk).  A group of LANES lanes takes one head at a time:
// lane l holds the NeoX pairs of elements [(c LANES + l) VEC, + VEC) and
// their partners hd/2 further, c < CH, so the rotation needs no exchange and
// the norm log2(LANES) shuffles.  A CTA's heads all belong to one token; a
// group takes `rounds` of them in turn.  Slots: q heads, k heads, v heads.
template <typename T, typename TO, int VEC, int LANES, int CH>
__global__ void __launch_bounds__(kNormThreads) norm_rope_append_kernel(const NormParams p)
{
    pdl_trigger();
    pdl_wait();  // inputs come from the previous kernel on the stream
    constexpr int kGroups = kNormThreads / LANES;
    const int i = blockIdx.x;
    const int hd = p.view.hd, half = hd / 2, hkv = p.view.hkv;
    const int q_heads = p.q ? p.hq : 0, slots = q_heads + 2 * hkv;
    const int lane = threadIdx.x % LANES;
    const int seq = p.seq_ids[i], pos = p.positions[i];
    if (seq == -1) return;  // a padding row
    if (seq < 0 || seq >= p.view.max_seqs || pos < 0 || pos >= p.view.capacity ||
        (p.table && pos >= p.table_max_pos)) {
        if (threadIdx.x == 0) record_status(p.status, HX_ERR_CAPACITY);
        return;
    }
    const int64_t off = token_offset(p.view, seq, 0, pos);
    if (off < 0 && threadIdx.x == 0) record_status(p.status, HX_ERR_CAPACITY);
    const float2* cs = p.table ? p.table + (int64_t)pos * half : nullptr;

    for (int round = 0; round < p.rounds; ++round) {
        const int slot = (blockIdx.y * p.rounds + round) * kGroups + (int)threadIdx.x / LANES;
        const bool live = slot < slots;
        const bool is_q = slot < q_heads, is_v = slot >= q_heads + hkv;
        const int h = is_q ? slot : is_v ? slot - q_heads - hkv : slot - q_heads;
        const T* src = is_q   ? static_cast<const T*>(p.q) + i * p.q_stride
                       : is_v ? static_cast<const T*>(p.v) + i * p.v_stride
                              : static_cast<const T*>(p.k) + i * p.k_stride;
        src += (int64_t)h * hd;
        float a[CH][VEC], b[CH][VEC];
        float ss = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int d = (c * LANES + lane) * VEC;
            if (live && d < half) {
                load_vec<T, VEC>(src + d, a[c]);
                load_vec<T, VEC>(src + d + half, b[c]);
#pragma unroll
                for (int e = 0; e < VEC; ++e) ss += a[c][e] * a[c][e] + b[c][e] * b[c][e];
            }
        }
#pragma unroll
        for (int o = LANES / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (!live) continue;
        const float r = 1.f / sqrtf(ss / (float)hd + p.eps);
        const T* w = static_cast<const T*>(is_q ? p.q_weight : p.k_weight);
        __half* dst = nullptr;
        if (!is_q && off >= 0)
            dst = reinterpret_cast<__half*>((is_v ? p.view.v : p.view.k) + off + h * p.view.head_stride);
        TO* qdst = static_cast<TO*>(p.q_out) + ((int64_t)i * p.hq + h) * hd;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int d = (c * LANES + lane) * VEC;
            if (d >= half) continue;
            if (!is_v) {
                float wa[VEC], wb[VEC];
                if (w) {
                    load_vec<T, VEC>(w + d, wa);
                    load_vec<T, VEC>(w + d + half, wb);
                }
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    float y1 = a[c][e] * r, y2 = b[c][e] * r;
                    if (w) {
                        y1 *= wa[e];
                        y2 *= wb[e];
                    }
                    if (cs) rotate(y1, y2, cs[d + e], y1, y2);
                    a[c][e] = y1;
                    b[c][e] = y2;
                }
            }
            if (is_q) {
                store_vec<TO, VEC>(qdst + d, a[c]);
                store_vec<TO, VEC>(qdst + d + half, b[c]);
            } else if (dst) {
                store_vec<__half, VEC>(dst + d, a[c]);
                store_vec<__half, VEC>(dst + d + half, b[c]);
            }
        }
    }
}

template <typename T, typename TO, int VEC, int LANES, int CH>
static int launch_norm(NormParams& p, int n, cudaStream_t s)
{
    constexpr int kGroups = kNormThreads / LANES;
    const int slots = (p.q ? p.hq : 0) + 2 * p.view.hkv;
    p.rounds = 1;
    const dim3 grid(n, (slots + kGroups * p.rounds - 1) / (kGroups * p.rounds));
    cudaError_t e = launch_kernel(norm_rope_append_kernel<T, TO, VEC, LANES, CH>, grid,
                                  dim3(kNormThreads), 0, s, true, p);
    if (e != cudaSuccess) return cuda_fail(e, "norm_rope_append_kernel launch");
    return check_launch("norm_rope_append_kernel");
}

// 16-byte accesses need every row, weight and head half to start on a 16-byte
// boundary; otherwise elements go one by one (four pairs a lane at most).
template <typename T, typename TO>
static int launch_norm_types(NormParams& p, int n, bool vec, cudaStream_t s)
{
    constexpr int VEC = 16 / sizeof(T);
    const int half = p.view.hd / 2;
    if (!vec) return launch_norm<T, TO, 1, 32, kMaxHeadDim / 64>(p, n, s);
    const int lanes = half / VEC;
    if (lanes <= 8) return launch_norm<T, TO, VEC, 8, 1>(p, n, s);
    if (lanes <= 16) return launch_norm<T, TO, VEC, 16, 1>(p, n, s);
    if constexpr (sizeof(T) == 4) return launch_norm<T, TO, VEC, 32, 1>(p, n, s);
    return fail(HX_ERR_UNSUPPORTED, "head_dim %d", p.view.hd);
}

}  // namespace hx

using namespace hx;

extern "C" int hx_norm_rope_append(hx_kv_cache* c, int layer, const void* q, int64_t q_stride,
                                   const void* k, int64_t k_stride, const void* v,
                                   int64_t v_stride, int dtype, const void* q_weight,
                                   const void* k_weight, float eps, const int32_t* seq_ids,
                                   const int32_t* positions, int n_tokens, int num_q_heads,
                                   const hx_rope_table* table, void* q_out, int q_out_dtype,
                                   hx_stream_t stream)
{
    HX_NVTX_RANGE("hx_norm_rope_append");
    if (!c) return fail(HX_ERR_INVALID, "null cache");
    if (layer < 0 || layer >= c->cfg.num_layers) return fail(HX_ERR_INVALID, "layer %d out of range", layer);
    if (n_tokens < 0) return fail(HX_ERR_INVALID, "n_tokens < 0");
    const int hd = c->cfg.head_dim, hkv = c->cfg.num_kv_heads;
    if ((q == nullptr) != (q_out == nullptr)) return fail(HX_ERR_INVALID, "q and q_out go together");
    if (q && (num_q_heads < hkv || num_q_heads % hkv))
        return fail(HX_ERR_INVALID, "num_q_heads %d must be a multiple of kv heads %d", num_q_heads, hkv);
    if (dtype != HX_FP16 && dtype != HX_FP32) return fail(HX_ERR_INVALID, "dtype %d", dtype);
    if (q && q_out_dtype != HX_FP16 && q_out_dtype != HX_FP32)
        return fail(HX_ERR_INVALID, "q_out dtype %d", q_out_dtype);
    if (!(eps >= 0.f)) return fail(HX_ERR_INVALID, "eps must be >= 0");
    if (table && table->cfg.head_dim != hd)
        return fail(HX_ERR_INVALID, "rope table head_dim %d != cache head_dim %d", table->cfg.head_dim, hd);
    if (n_tokens == 0) return HX_OK;
    if (!k || !v || !seq_ids || !positions) return fail(HX_ERR_INVALID, "null k/v/seq_ids/positions");
    if (n_tokens > 1 && ((q && q_stride < (int64_t)num_q_heads * hd) || k_stride < (int64_t)hkv * hd ||
                         v_stride < (int64_t)hkv * hd))
        return fail(HX_ERR_INVALID, "a row stride is shorter than its row");
    if (int rc = check_device(c->device, "the cache")) return rc;
    if (table)
        if (int rc = check_device(table->device, "the rope table")) return rc;

    NormParams p{};
    p.view = make_view(c, layer);
    p.q = q;
    p.k = k;
    p.v = v;
    p.q_stride = q_stride;
    p.k_stride = k_stride;
    p.v_stride = v_stride;
    p.q_weight = q_weight;
    p.k_weight = k_weight;
    p.seq_ids = seq_ids;
    p.positions = positions;
    p.table = table ? table->d_cos_sin : nullptr;
    p.table_max_pos = table ? table->cfg.max_pos : 0;
    p.q_out = q_out;
    p.hq = q ? num_q_heads : 0;
    p.eps = eps;
    p.status = status_word();
    const int es = dtype == HX_FP16 ? 2 : 4;
    auto at16 = [](const void* ptr) { return reinterpret_cast<uintptr_t>(ptr) % 16 == 0; };
    auto rows16 = [&](const void* ptr, int64_t stride) { return at16(ptr) && (n_tokens == 1 || stride * es % 16 == 0); };
    const bool vec = (hd / 2) % (16 / es) == 0 && (!q || rows16(q, q_stride)) && rows16(k, k_stride) &&
                     rows16(v, v_stride) && at16(q_out) && at16(q_weight) && at16(k_weight);
    cudaStream_t s = (cudaStream_t)stream;
    const bool q32 = q && q_out_dtype == HX_FP32;
    if (dtype == HX_FP16)
        return q32 ? launch_norm_types<__half, float>(p, n_tokens, vec, s)
                   : launch_norm_types<__half, __half>(p, n_tokens, vec, s);
    return q32 ? launch_norm_types<float, float>(p, n_tokens, vec, s)
               : launch_norm_types<float, __half>(p, n_tokens, vec, s);
}
