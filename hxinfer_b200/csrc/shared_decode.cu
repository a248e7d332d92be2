// shared_decode.cu — decode attention of a batch whose sequences begin with
// the same positions (hx_kv_share): the prefix is read once for all of them.
//
//   o_i = softmax(scale q_i [K_P ; K_i]^T) [V_P ; V_i]
//
// with K_P, V_P positions [0, prefix_len) of prefix_seq and K_i, V_i positions
// [prefix_len, lengths[i]) of sequence i.
#include <algorithm>
#include <cmath>

#include "hx_common.cuh"

namespace hx {

struct SharedParams {
    KVView view;
    const __half* q;            // [n_seqs][hq * hd]
    const int32_t* seq_ids;
    const int32_t* lengths;
    int n_seqs, hq, group, prefix_seq, prefix_len;
    float scale_log2;
    void* out;
    int out_f32;
    int* status;
};

// What a row of the batch is: its sequence, and its length or 0 for a row of
// zeros, or -1 for padding.  Only one thread of a call records the errors.
__device__ __forceinline__ int row_length(const SharedParams& p, int s, bool record)
{
    const int seq = p.seq_ids[s], len = p.lengths[s];
    if (seq == -1) return -1;
    if (len == 0) return 0;
    if (seq < 0 || seq >= p.view.max_seqs || len < p.prefix_len || len < 0 || len > p.view.capacity) {
        if (record) record_status(p.status, HX_ERR_CAPACITY);
        return 0;
    }
    return len;
}

// Any head_dim (<= 256) and group: one CTA of four warps per (sequence, q
// head); warps take positions in turn, lanes dims; online softmax; the warps
// merge in shared memory.
__global__ void __launch_bounds__(128) shared_generic_kernel(const SharedParams p)
{
    const int s = blockIdx.x / p.hq, qh = blockIdx.x % p.hq;
    const int kvh = qh / p.group;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const KVView& v = p.view;
    const int hd = v.hd;
    const int len = row_length(p, s, threadIdx.x == 0);
    if (len < 0) return;
    constexpr int kPer = kMaxHeadDim / 32;
    float qv[kPer], acc[kPer];
    const int64_t qoff = ((int64_t)s * p.hq + qh) * hd;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        const int d = lane + 32 * e;
        acc[e] = 0.f;
        qv[e] = d < hd ? __half2float(p.q[qoff + d]) : 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int pos = warp; pos < len; pos += 4) {
        const int64_t off = token_offset(v, pos < p.prefix_len ? p.prefix_seq : p.seq_ids[s], kvh, pos);
        if (off < 0) {
            record_status(p.status, HX_ERR_CAPACITY);
            break;
        }
        const __half* kr = reinterpret_cast<const __half*>(v.k + off);
        const __half* vr = reinterpret_cast<const __half*>(v.v + off);
        float dot = 0.f;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            const int d = lane + 32 * e;
            if (d < hd) dot += qv[e] * __half2float(kr[d]);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        const float sc = dot * p.scale_log2;
        const float mn = fmaxf(m, sc);
        const float mu = mn == -INFINITY ? 0.f : mn;
        const float al = fast_exp2(m - mu), pr = fast_exp2(sc - mu);
        l = l * al + pr;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            const int d = lane + 32 * e;
            acc[e] = acc[e] * al + (d < hd ? pr * __half2float(vr[d]) : 0.f);
        }
        m = mn;
    }
    __shared__ float sm_m[4], sm_l[4], sm_o[4][kMaxHeadDim];
    if (lane == 0) {
        sm_m[warp] = m;
        sm_l[warp] = l;
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        const int d = lane + 32 * e;
        if (d < hd) sm_o[warp][d] = acc[e];
    }
    __syncthreads();
    const float M = fmaxf(fmaxf(sm_m[0], sm_m[1]), fmaxf(sm_m[2], sm_m[3]));
    const float Mu = M == -INFINITY ? 0.f : M;
    for (int d = threadIdx.x; d < hd; d += blockDim.x) {
        float L = 0.f, o = 0.f;
        for (int w = 0; w < 4; ++w) {
            const float wgt = fast_exp2(sm_m[w] - Mu);
            L += wgt * sm_l[w];
            o += wgt * sm_o[w][d];
        }
        const float val = len > 0 ? o / L : 0.f;
        if (p.out_f32) static_cast<float*>(p.out)[qoff + d] = val;
        else static_cast<__half*>(p.out)[qoff + d] = __float2half_rn(val);
    }
}

static size_t shared_ws_bytes(const hx_kv_cache*, int, int, int) { return 16; }

}  // namespace hx

using namespace hx;

extern "C" size_t hx_decode_shared_workspace_bytes(const hx_kv_cache* c, int n_seqs, int num_q_heads,
                                                   int prefix_len)
{
    if (!c || n_seqs < 1 || num_q_heads < c->cfg.num_kv_heads || prefix_len < 0) return 0;
    return shared_ws_bytes(c, n_seqs, num_q_heads, prefix_len);
}

extern "C" int hx_decode_attention_shared(const hx_kv_cache* c, int layer, const void* q,
                                          const int32_t* seq_ids, const int32_t* lengths, int n_seqs,
                                          int num_q_heads, int prefix_seq, int prefix_len, float scale,
                                          void* out, int out_dtype, void* workspace,
                                          size_t workspace_bytes, hx_stream_t stream)
{
    HX_NVTX_RANGE("hx_decode_attention_shared");
    if (!c) return fail(HX_ERR_INVALID, "null cache");
    if (layer < 0 || layer >= c->cfg.num_layers) return fail(HX_ERR_INVALID, "layer %d out of range", layer);
    if (n_seqs < 0) return fail(HX_ERR_INVALID, "n_seqs < 0");
    const int hkv = c->cfg.num_kv_heads;
    if (num_q_heads < hkv || num_q_heads % hkv)
        return fail(HX_ERR_INVALID, "num_q_heads %d must be a multiple of kv heads %d", num_q_heads, hkv);
    if (out_dtype != HX_FP16 && out_dtype != HX_FP32) return fail(HX_ERR_INVALID, "out dtype %d", out_dtype);
    if (!(scale > 0.f) || std::isinf(scale)) return fail(HX_ERR_INVALID, "scale must be positive and finite");
    if (prefix_len < 0) return fail(HX_ERR_INVALID, "prefix_len < 0");
    if (prefix_seq < 0 || prefix_seq >= c->cfg.max_seqs)
        return fail(HX_ERR_INVALID, "prefix_seq %d out of range", prefix_seq);
    if (prefix_len > c->cfg.max_tokens_per_seq || (int64_t)prefix_len > (int64_t)c->n_mapped[prefix_seq] * kBlockTokens)
        return fail(HX_ERR_CAPACITY, "prefix_seq %d does not hold %d positions", prefix_seq, prefix_len);
    if (n_seqs == 0) return HX_OK;
    if (!q || !seq_ids || !lengths || !out) return fail(HX_ERR_INVALID, "null q/seq_ids/lengths/out");
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15)
        return fail(HX_ERR_INVALID, "q and out must be 16-byte aligned");
    if ((int64_t)n_seqs * num_q_heads > INT32_MAX)
        return fail(HX_ERR_INVALID, "%d sequences of %d q heads are too many", n_seqs, num_q_heads);
    const size_t need = shared_ws_bytes(c, n_seqs, num_q_heads, prefix_len);
    if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15))
        return fail(HX_ERR_INVALID, "workspace of %zu bytes (16-byte aligned) needed, have %zu", need,
                    workspace ? workspace_bytes : 0);
    if (int rc = check_device(c->device, "the cache")) return rc;
    SharedParams p{};
    p.view = make_view(c, layer);
    p.q = (const __half*)q;
    p.seq_ids = seq_ids;
    p.lengths = lengths;
    p.n_seqs = n_seqs;
    p.hq = num_q_heads;
    p.group = num_q_heads / hkv;
    p.prefix_seq = prefix_seq;
    p.prefix_len = prefix_len;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.out = out;
    p.out_f32 = out_dtype == HX_FP32;
    p.status = status_word();
    shared_generic_kernel<<<n_seqs * num_q_heads, 128, 0, (cudaStream_t)stream>>>(p);
    return check_launch("shared_generic_kernel");
}
