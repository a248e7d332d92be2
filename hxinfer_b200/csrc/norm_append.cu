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
// Each element is read and written once with a dozen operations, so the bound
// is HBM for prompts and the chain of dependent loads (position, block table,
// table row) for decode batches.  Measured: 8192 tokens of 32 + 8 + 8 heads of
// 128 in fp16 (206 MB) 52 us, 4.0 TB/s; what keeps it from HBM's rate is the
// short life of its CTAs and the chain in each (a plain copy of the same bytes
// takes 32 us).  64 tokens 2.4 us and one 2.0 us in a graph, of which 1.7
// are the launch; the caller's side of a call is longer, 8 us from Python.
#include <algorithm>

#include "hx_common.cuh"

namespace hx {

constexpr int kNormThreads = 128;

// VEC elements as they lie in memory: 16 bytes, or one element.
template <typename T, int VEC>
struct RawVec {
    T v[VEC];
};
template <>
struct __align__(16) RawVec<__half, 8> {
    __half v[8];
};
template <>
struct __align__(16) RawVec<float, 4> {
    float v[4];
};

template <typename T, int VEC>
__device__ __forceinline__ RawVec<T, VEC> load_raw(const T* p)
{
    return *reinterpret_cast<const RawVec<T, VEC>*>(p);
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
    int table_max_pos, hq, n;
    float eps, inv_hd;
    int* status;
};

// A group of LANES lanes takes one head at a time: lane l holds the NeoX pairs
// of elements [(c LANES + l) VEC, + VEC) and their partners hd/2 further,
// c < CH, so the rotation needs no exchange and the norm log2(LANES) shuffles.
// A CTA's heads all belong to one token; a group takes HEADS of them, loaded
// together, which then share the lane's table row.  Slots: q heads, k heads, v
// heads.  grid (slot chunk, token).
template <typename T, typename TO, int VEC, int LANES, int CH, int HEADS>
__global__ void __launch_bounds__(kNormThreads) norm_rope_append_kernel(const NormParams p)
{
    pdl_wait();     // inputs come from the previous kernel on the stream
    pdl_trigger();  // not before: a dependent may read early what kernels before this one wrote
    constexpr int kGroups = kNormThreads / LANES;
    const int hd = p.view.hd, half = hd / 2, hkv = p.view.hkv;
    const int q_heads = p.q ? p.hq : 0, slots = q_heads + 2 * hkv;
    const int lane = threadIdx.x % LANES;
    for (int i = blockIdx.y; i < p.n; i += gridDim.y) {
        const int seq = p.seq_ids[i], pos = p.positions[i];
        RawVec<T, VEC> a[HEADS][CH], b[HEADS][CH];
#pragma unroll
        for (int j = 0; j < HEADS; ++j) {
            const int slot = (blockIdx.x * HEADS + j) * kGroups + (int)threadIdx.x / LANES;
            const T* src = slot < q_heads
                ? static_cast<const T*>(p.q) + i * p.q_stride + (int64_t)slot * hd
                : slot < q_heads + hkv
                    ? static_cast<const T*>(p.k) + i * p.k_stride + (int64_t)(slot - q_heads) * hd
                    : static_cast<const T*>(p.v) + i * p.v_stride + (int64_t)(slot - q_heads - hkv) * hd;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int d = (c * LANES + lane) * VEC;
                if (slot < slots && d < half) {  // whatever the position: its loads run beside these
                    a[j][c] = load_raw<T, VEC>(src + d);
                    b[j][c] = load_raw<T, VEC>(src + d + half);
                } else {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) a[j][c].v[e] = b[j][c].v[e] = T(0.f);
                }
            }
        }
        if (seq == -1) continue;  // a padding row
        if (seq < 0 || seq >= p.view.max_seqs || pos < 0 || pos >= p.view.capacity ||
            (p.table && pos >= p.table_max_pos)) {
            if (threadIdx.x == 0) record_status(p.status, HX_ERR_CAPACITY);
            continue;
        }
        // An unmapped block shows beside the table row's loads and only stops the
        // stores (leaving here makes 8192 tokens take 62 us instead of 52).
        const int64_t off = token_offset(p.view, seq, 0, pos);
        if (off < 0 && threadIdx.x == 0) record_status(p.status, HX_ERR_CAPACITY);
        float2 cs[CH][VEC];
        if (p.table) {
            const float2* row = p.table + (int64_t)pos * half;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int d = (c * LANES + lane) * VEC;
                if (d >= half) continue;
                if constexpr (VEC == 1) {
                    cs[c][0] = row[d];
                } else {
#pragma unroll
                    for (int e = 0; e < VEC; e += 2) {
                        const float4 two = *reinterpret_cast<const float4*>(row + d + e);
                        cs[c][e] = make_float2(two.x, two.y);
                        cs[c][e + 1] = make_float2(two.z, two.w);
                    }
                }
            }
        }
#pragma unroll
        for (int j = 0; j < HEADS; ++j) {
            const int slot = (blockIdx.x * HEADS + j) * kGroups + (int)threadIdx.x / LANES;
            const bool is_q = slot < q_heads, is_v = slot >= q_heads + hkv;
            const int h = is_q ? slot : is_v ? slot - q_heads - hkv : slot - q_heads;
            float ss = 0.f;
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float x = (float)a[j][c].v[e], y = (float)b[j][c].v[e];
                    ss = fmaf(x, x, fmaf(y, y, ss));
                }
#pragma unroll
            for (int o = LANES / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (slot >= slots) continue;
            const float r = rsqrtf(fmaf(ss, p.inv_hd, p.eps));  // off by 2 ulp at most
            const T* w = static_cast<const T*>(is_q ? p.q_weight : p.k_weight);
            __half* dst = nullptr;
            if (!is_q && off >= 0)
                dst = reinterpret_cast<__half*>((is_v ? p.view.v : p.view.k) + off + h * p.view.head_stride);
            TO* qdst = static_cast<TO*>(p.q_out) + ((int64_t)i * p.hq + h) * hd;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int d = (c * LANES + lane) * VEC;
                if (d >= half) continue;
                float ya[VEC], yb[VEC];
                if (is_v) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        ya[e] = (float)a[j][c].v[e];
                        yb[e] = (float)b[j][c].v[e];
                    }
                } else {
                    RawVec<T, VEC> wa, wb;
                    if (w) {
                        wa = load_raw<T, VEC>(w + d);
                        wb = load_raw<T, VEC>(w + d + half);
                    }
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        float y1 = (float)a[j][c].v[e] * r, y2 = (float)b[j][c].v[e] * r;
                        if (w) {
                            y1 *= (float)wa.v[e];
                            y2 *= (float)wb.v[e];
                        }
                        ya[e] = y1;
                        yb[e] = y2;
                        if (p.table) {
                            ya[e] = fmaf(y1, cs[c][e].x, -(y2 * cs[c][e].y));
                            yb[e] = fmaf(y2, cs[c][e].x, y1 * cs[c][e].y);
                        }
                    }
                }
                if (is_q) {
                    if (off >= 0) {
                        store_vec<TO, VEC>(qdst + d, ya);
                        store_vec<TO, VEC>(qdst + d + half, yb);
                    }
                } else if (dst) {
                    store_vec<__half, VEC>(dst + d, ya);
                    store_vec<__half, VEC>(dst + d + half, yb);
                }
            }
        }
    }
}

template <typename T, typename TO, int VEC, int LANES, int CH, int HEADS>
static int launch_norm_heads(const NormParams& p, int n, cudaStream_t s)
{
    constexpr int kGroups = kNormThreads / LANES;
    const int slots = (p.q ? p.hq : 0) + 2 * p.view.hkv;
    const dim3 grid((slots + kGroups * HEADS - 1) / (kGroups * HEADS), std::min(n, 65535));
    cudaError_t e = launch_kernel(norm_rope_append_kernel<T, TO, VEC, LANES, CH, HEADS>, grid, dim3(kNormThreads), 0, s,
                                  true, p);
    if (e != cudaSuccess) return cuda_fail(e, "norm_rope_append_kernel launch");
    return check_launch("norm_rope_append_kernel");
}

// Two heads a group when one each would be several times what the GPU holds at
// once (8192 tokens, 32 + 8 + 8 heads of 128: 52 us with two, 59 with one, 57
// with three; 64 tokens fit at once: 2.8 to 3.0 us either way).
template <typename T, typename TO, int VEC, int LANES, int CH>
static int launch_norm(const NormParams& p, int n, cudaStream_t s)
{
    const int64_t heads = (int64_t)n * ((p.q ? p.hq : 0) + 2 * p.view.hkv);
    if constexpr (CH == 1)
        if (heads * LANES > (int64_t)num_sms() * 2048) return launch_norm_heads<T, TO, VEC, LANES, CH, 2>(p, n, s);
    return launch_norm_heads<T, TO, VEC, LANES, CH, 1>(p, n, s);
}

// 16-byte accesses need every row, weight and head half to start on a 16-byte
// boundary; otherwise elements go one by one (four pairs a lane at most).
template <typename T, typename TO>
static int launch_norm_types(const NormParams& p, int n, bool vec, cudaStream_t s)
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

extern "C" int hx_norm_rope_append(hx_kv_cache* c, int layer, const hx_norm_append_spec* spec,
                                   hx_stream_t stream)
{
    HX_NVTX_RANGE("hx_norm_rope_append");
    if (!c) return fail(HX_ERR_INVALID, "null cache");
    if (!spec) return fail(HX_ERR_INVALID, "null spec");
    if (layer < 0 || layer >= c->cfg.num_layers) return fail(HX_ERR_INVALID, "layer %d out of range", layer);
    const hx_norm_append_spec& a = *spec;
    if (a.n_tokens < 0) return fail(HX_ERR_INVALID, "n_tokens < 0");
    const int hd = c->cfg.head_dim, hkv = c->cfg.num_kv_heads;
    if ((a.q == nullptr) != (a.q_out == nullptr)) return fail(HX_ERR_INVALID, "q and q_out go together");
    if (a.q && (a.num_q_heads < hkv || a.num_q_heads % hkv))
        return fail(HX_ERR_INVALID, "num_q_heads %d must be a multiple of kv heads %d", a.num_q_heads, hkv);
    if (a.dtype != HX_FP16 && a.dtype != HX_FP32) return fail(HX_ERR_INVALID, "dtype %d", a.dtype);
    if (a.q && a.q_out_dtype != HX_FP16 && a.q_out_dtype != HX_FP32)
        return fail(HX_ERR_INVALID, "q_out dtype %d", a.q_out_dtype);
    if (!(a.eps >= 0.f)) return fail(HX_ERR_INVALID, "eps must be >= 0");
    if (a.table && a.table->cfg.head_dim != hd)
        return fail(HX_ERR_INVALID, "rope table head_dim %d != cache head_dim %d", a.table->cfg.head_dim, hd);
    if (a.n_tokens == 0) return HX_OK;
    if (!a.k || !a.v || !a.seq_ids || !a.positions) return fail(HX_ERR_INVALID, "null k/v/seq_ids/positions");
    if (a.n_tokens > 1 && ((a.q && a.q_stride < (int64_t)a.num_q_heads * hd) || a.k_stride < (int64_t)hkv * hd ||
                           a.v_stride < (int64_t)hkv * hd))
        return fail(HX_ERR_INVALID, "a row stride is shorter than its row");
    if (int rc = check_device(c->device, "the cache")) return rc;
    if (a.table)
        if (int rc = check_device(a.table->device, "the rope table")) return rc;

    NormParams p{};
    p.view = make_view(c, layer);
    p.q = a.q;
    p.k = a.k;
    p.v = a.v;
    p.q_stride = a.q_stride;
    p.k_stride = a.k_stride;
    p.v_stride = a.v_stride;
    p.q_weight = a.q_weight;
    p.k_weight = a.k_weight;
    p.seq_ids = a.seq_ids;
    p.positions = a.positions;
    p.table = a.table ? a.table->d_cos_sin : nullptr;
    p.table_max_pos = a.table ? a.table->cfg.max_pos : 0;
    p.q_out = a.q_out;
    p.hq = a.q ? a.num_q_heads : 0;
    p.n = a.n_tokens;
    p.eps = a.eps;
    p.inv_hd = 1.f / (float)hd;
    p.status = status_word();
    const int es = a.dtype == HX_FP16 ? 2 : 4;
    auto at16 = [](const void* ptr) { return reinterpret_cast<uintptr_t>(ptr) % 16 == 0; };
    auto rows16 = [&](const void* ptr, int64_t stride) { return at16(ptr) && (a.n_tokens == 1 || stride * es % 16 == 0); };
    const bool vec = (hd / 2) % (16 / es) == 0 && (!a.q || rows16(a.q, a.q_stride)) && rows16(a.k, a.k_stride) &&
                     rows16(a.v, a.v_stride) && at16(a.q_out) && at16(a.q_weight) && at16(a.k_weight);
    cudaStream_t s = (cudaStream_t)stream;
    const bool q32 = a.q && a.q_out_dtype == HX_FP32;
    if (a.dtype == HX_FP16)
        return q32 ? launch_norm_types<__half, float>(p, a.n_tokens, vec, s)
                   : launch_norm_types<__half, __half>(p, a.n_tokens, vec, s);
    return q32 ? launch_norm_types<float, float>(p, a.n_tokens, vec, s)
               : launch_norm_types<float, __half>(p, a.n_tokens, vec, s);
}
