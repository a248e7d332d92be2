// shared_decode.cu — decode attention of a batch whose sequences begin with
// the same positions (hx_kv_share): the prefix is read once for all of them.
//
//   o_i = softmax(scale q_i [K_P ; K_i]^T) [V_P ; V_i]
//
// with K_P, V_P positions [0, prefix_len) of prefix_seq and K_i, V_i positions
// [prefix_len, lengths[i]) of sequence i.  Softmax over a concatenation splits
// into partial results (O, m, l) over parts of the keys, merged by
//   M = max m,  o = sum 2^(m - M) O / sum 2^(m - M) l.
//
// Prefix: the q rows of all sequences that read one kv head (sequence by
// sequence, the head's group of q heads within) are stacked into tiles of up
// to 128 rows, so one tile of keys serves 128 rows on the tcgen05 tensor cores
// (M = 128 rows, N = 128 keys), as in causal prefill but without its mask:
// 4 * 128 * 128 * 128 operations per 64 KB of K and V.
//
// Suffix: every sequence has its own keys, so only the rows of one sequence
// and kv head (a segment; 16 rows at most, larger groups make several) share
// them.  A warp takes a run of 32-key steps by itself, through a ring of its
// own that TMA fills.  The products run on mma.sync with the keys as M and the
// rows as N, as in hx_decode_attention.  No warp waits for another, and short
// suffixes cost what they hold; bound by HBM.
//
// One launch does both.  Of the CTAs, one per SM, the first n_pre share the
// prefix tiles (row tile by row tile, keys in order) evenly, and the warps of
// the others the suffix steps (sequence by sequence, head by head), with n_pre
// weighed so that both parts end together: the tensor cores of some SMs work
// while others stream.  Each piece (a CTA's part of one row tile, a warp's
// part of one segment) leaves its partial result in the workspace, and
// shared_combine_kernel merges them.
//
// Slots of partial results: a piece that begins with the first tile (step) of
// segment s takes slot s, and one that begins inside a segment (only a CTA's
// or warp's first piece can) takes slot n_segments + its CTA (warp) number.
//
// What bounds it: a prefix tile takes 1.1 us alone and 1.5 when all SMs load,
// twice its products at the dense rate: a product of 128 rows by 16 takes some
// 100 cycles for up to 128 columns (64 at the dense rate), and the tensor cores
// and the softmax wait for each other at the two buffers.  Sharing K and V
// between two row tiles and giving each warpgroup tiles of its own were tried
// under an earlier split of the CTAs (64, 32768: 76 us in a graph, 78 without at
// that time, 68 since; the others 2 to 8 us slower cold); not tried again under
// the present one.  A suffix step of eight warps takes 0.26 us, 64 GB/s of an SM.
// Launches, plan and combine add 6 us.  Measured in a graph (q heads / kv heads,
// own positions up to 1,024), and per call from Python with a cold L2: 8
// sequences, prefix 2048, 28 / 4: 13.6 us (14.1); 64, 8192, 32 / 8: 32.9 (36.0);
// 64, 32768, 32 / 8: 68.5 (80; 509 Tflop/s in a graph); 33, 5001, 32 / 32: 40.4
// (45.8; 4.3 TB/s).
//
// All of this is for head_dim 128 and groups of up to 128 q heads.  Other calls
// take shared_generic_kernel, a CTA per sequence and q head, which reads the
// prefix once for each.
#include <algorithm>
#include <cmath>

#include "hx_split.h"
#include "hx_tcgen05.cuh"

namespace hx {

constexpr int kShSoftmaxWarps = 8;
constexpr int kShProducerWarp = 8, kShMmaWarp = 9;
constexpr int kShThreads = 32 * 10;
constexpr int kShRows = 128, kShKeys = 128;      // prefix tile
constexpr int kShRegion = 128 * 128;             // 128 rows x 64 fp16, one swizzled region
constexpr int kShStages = 3;                     // prefix K and V rings
constexpr int kShSufKeys = 32;                   // keys of a suffix step
constexpr int kShSufRing = 3;                    // a warp's ring: steps' K and V in turn
constexpr int kShSufBox = kShSufKeys * 128;      // one 64 x 32 box
constexpr int kShSufSlot = 2 * kShSufBox;        // K or V of a step
constexpr int kShSufMinSteps = 2;                // fewer are not worth a warp's partial result
// Costs to a CTA in units of a suffix step of eight warps (0.26 us on a busy
// GPU): a prefix tile, what a piece takes besides its tiles, and a segment's
// start and end.  A tile at 4 to 5 gives the same times; at 6, 64 sequences
// behind 32768 positions take 77.8 us instead of 68.1, 33 behind 5001 42.8
// instead of 40.4.
constexpr float kShPrefixCost = 4.75f, kShPieceCost = 16.f, kShSegmentCost = 2.f;

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
    // fast path
    int seqs_per_tile;          // sequences stacked in a row tile
    int row_tiles;              // per kv head
    int chunk, chunks;          // q rows of a suffix segment, and segments per (sequence, kv head)
    int key_tiles;              // 128-key tiles of the prefix
    int ctas;                   // CTAs launched
    float* pre_o;               // [slots][32 chunks][128 rows][4]: rows beside each other
    float2* pre_ml;             // [slots][128]
    float* suf_o;               // [slots][chunk][128]
    float2* suf_ml;             // [slots][chunk]
};

// What a row of the batch is: its length, 0 for a row of zeros, or -1 for
// padding.
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

// 32-key steps of a sequence's own keys, from the one that holds prefix_len.
__device__ __forceinline__ int suffix_steps(const SharedParams& p, int len)
{
    return len > p.prefix_len ? (len - 1) / kShSufKeys - p.prefix_len / kShSufKeys + 1 : 0;
}

// How the work is cut: prefix tiles [n_pre c / pre, n_pre (c + 1) / pre) go to
// CTA c < pre, and suffix steps [n_suf k / suf, n_suf (k + 1) / suf) to warp k
// of the other CTAs, numbered CTA by CTA within each warp position, so that
// few warps spread over all of them.
struct SharedPlan {
    int64_t n_pre, n_suf;  // tiles, steps
    int pre, suf;          // CTAs, warps

    // By a whole warp: its lanes weigh 32 splits around the one that the costs
    // suggest, half of them with as many CTAs for every row tile (ranges that
    // line up with the row tiles spare their CTAs a second piece).
    __device__ SharedPlan(const SharedParams& p, int64_t steps_per_segment, int lane)
    {
        const int64_t segs = (int64_t)p.view.hkv * p.row_tiles;
        n_pre = segs * p.key_tiles;
        n_suf = steps_per_segment * p.view.hkv * p.chunks;
        pre = n_suf == 0 ? p.ctas : 0;
        if (n_suf > 0 && n_pre > 0) {
            const float tiles = (float)n_pre, rows = (float)segs;
            const float suffix = (float)n_suf + kShSegmentCost * (float)p.n_seqs * p.view.hkv * p.chunks;
            const float prefix = tiles * kShPrefixCost + rows * kShPieceCost;
            const float share = (float)p.ctas * (prefix / (prefix + suffix));
            const int even = lane < 16 ? (int)min((float)p.ctas, (rintf(share / rows) + (float)(lane - 8)) * rows)
                                       : (int)share + 2 * (lane - 24);
            const int c = max(1, min(p.ctas - 1, even));
            const float per = (float)c / rows;
            const float pieces = per == floorf(per) ? 1.f : 2.f + floorf(1.f / per);
            const float t = fmaxf(ceilf(tiles / (float)c) * kShPrefixCost + pieces * kShPieceCost,
                                  suffix / (float)(p.ctas - c));
            // the least time, in 2^-14 of a perfect split's, then the fewest CTAs
            const float rel = t * (float)p.ctas / (prefix + suffix) * 16384.f;
            const unsigned key = (unsigned)fminf(rel, 2e6f) << 11 | min((unsigned)c, 0x7ffu);
            pre = (int)(__reduce_min_sync(0xffffffffu, key) & 0x7ffu);
        }
        if (pre > n_pre) pre = (int)n_pre;
        suf = (p.ctas - pre) * kShSoftmaxWarps;
        const int64_t most = (n_suf + kShSufMinSteps - 1) / kShSufMinSteps;
        if (suf > most) suf = (int)most;
    }
};

// Position in the list of suffix steps.
struct SuffixCursor {
    int s, h, rc, j, steps, len, seq;

    __device__ void load(const SharedParams& p, int seq_slot)
    {
        s = seq_slot;
        steps = 0;
        if (s >= p.n_seqs) return;
        len = row_length(p, s, false);
        steps = suffix_steps(p, len);
        seq = p.seq_ids[s];
    }
    __device__ void next(const SharedParams& p)
    {
        if (++j < steps) return;
        j = 0;
        if (++rc < p.chunks) return;
        rc = 0;
        if (++h < p.view.hkv) return;
        h = 0;
        do load(p, s + 1);
        while (steps == 0 && s < p.n_seqs);
    }
    __device__ int64_t segment(const SharedParams& p) const
    {
        return ((int64_t)s * p.view.hkv + h) * p.chunks + rc;
    }
};

struct SharedSmem {
    uint8_t q[2][kShRegion];                     // [d half]
    // prefix: K ring [stage][d half] then V ring; suffix: the warps' rings
    uint8_t ring[2 * kShStages][2][kShRegion];
    uint64_t q_full;
    uint64_t k_full[kShStages], k_empty[kShStages];
    uint64_t v_full[kShStages], v_empty[kShStages];
    uint64_t s_full[2];                          // per TMEM S/P buffer
    uint64_t p_full[2][2], pv_done[2][2];        // [key half][TMEM S/P buffer]
    uint64_t mma_idle;
    uint32_t tmem_base;
    int abort_flag;
    int64_t pre0, pre1;                          // this CTA's prefix tiles (not in registers: the softmax needs them)
    uint64_t suf_full[kShSoftmaxWarps][kShSufRing];
};
static_assert(kShSoftmaxWarps * kShSufRing * kShSufSlot <= 2 * kShStages * 2 * kShRegion, "the rings share bytes");

// Warp-wide inclusive sum.
__device__ __forceinline__ int64_t warp_sum_incl(int64_t v, int lane)
{
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += y;
    }
    return v;
}

// The sequences' suffix steps, a warp's lane holding those of sequences
// lane, lane + 32, ...: the first four rounds are loaded together and kept, so
// a call of up to 128 sequences plans with one round of loads.
struct SeqSteps {
    static constexpr int kKept = 4;
    int kept[kKept];

    __device__ SeqSteps(const SharedParams& p, int lane, bool record)
    {
#pragma unroll
        for (int r = 0; r < kKept; ++r) kept[r] = load(p, 32 * r + lane, record);
    }
    static __device__ int load(const SharedParams& p, int s, bool record)
    {
        return s < p.n_seqs ? suffix_steps(p, row_length(p, s, record)) : 0;
    }
    __device__ int get(const SharedParams& p, int base, int lane, bool record) const
    {
        int v = 0;
#pragma unroll
        for (int r = 0; r < kKept; ++r)
            if (base == 32 * r) v = kept[r];
        return base >= 32 * kKept ? load(p, base + lane, record) : v;
    }
    // Steps of a segment summed over all sequences, and over those before `s`
    // (each lane's own).
    __device__ int64_t total(const SharedParams& p, int lane, int s, int64_t* before, bool record) const
    {
        int64_t sum = 0;
        for (int base = 0; base < p.n_seqs; base += 32) {
            const int t = get(p, base, lane, record);
            const int64_t incl = warp_sum_incl(t, lane);
            if (before) {
                const int64_t excl = __shfl_sync(0xffffffffu, incl - t, s & 31);
                if (s >> 5 == base >> 5) *before = sum + excl;
            }
            sum += __shfl_sync(0xffffffffu, incl, 31);
        }
        return sum;
    }
    // The cursor at suffix step `item`.
    __device__ SuffixCursor find(const SharedParams& p, int lane, int64_t item) const
    {
        const int per = p.view.hkv * p.chunks;  // segments of a sequence
        SuffixCursor cur{p.n_seqs, 0, 0, 0, 0, 0, 0};
        int64_t run = 0;
        for (int base = 0; base < p.n_seqs; base += 32) {
            const int64_t t = (int64_t)get(p, base, lane, false) * per;
            const int64_t incl = warp_sum_incl(t, lane);
            const unsigned hit = __ballot_sync(0xffffffffu, run + incl > item);
            if (hit) {
                const int src = __ffs(hit) - 1;
                const unsigned off = (unsigned)(item - run - __shfl_sync(0xffffffffu, incl - t, src));
                cur.load(p, base + src);
                const int seg = off / cur.steps;
                cur.j = off % cur.steps;
                cur.h = seg / p.chunks;
                cur.rc = seg % p.chunks;
                break;
            }
            run += __shfl_sync(0xffffffffu, incl, 31);
        }
        return cur;
    }
};

// ------------------------------------------------------------------ prefix

// One row tile of a piece: q rows of sequences [s0, s0 + seqs_per_tile) for kv
// head h over key tiles [j0, j0 + nk); `done` counts the key tiles of the
// CTA's earlier pieces, which the barriers' phases go on from.
struct PrefixPiece {
    int h, rt, j0, nk;
    int64_t slot;
    int done, index;
};

__device__ __forceinline__ bool sh_wait(const SharedParams& p, SharedSmem& sm, uint64_t* bar, uint32_t parity)
{
    return mbar_wait_or_abort(&sm.abort_flag, bar, parity, p.status);
}

// lane 0: Q and the K ring, lane 1: the V ring (as in causal prefill).
__device__ void prefix_producer(const SharedParams& p, SharedSmem& sm, const PrefixPiece& pc,
                                const CUtensorMap* tm_q, const CUtensorMap* tm_k, const CUtensorMap* tm_v, int lane)
{
    const uint64_t pol = l2_evict_last_policy();  // the other row tiles read the keys again
    const KVView& v = p.view;
    const bool is_k = lane == 0;
    uint64_t* fulls = is_k ? sm.k_full : sm.v_full;
    uint64_t* empties = is_k ? sm.k_empty : sm.v_empty;
    if (is_k) {
        const int s0 = pc.rt * p.seqs_per_tile;
        mbar_arrive_expect_tx(&sm.q_full, 256 * p.seqs_per_tile * p.group);
        tma_load_3d(sm.q[0], tm_q, 0, pc.h * p.group, s0, &sm.q_full, pol);
        tma_load_3d(sm.q[1], tm_q, 64, pc.h * p.group, s0, &sm.q_full, pol);
    }
    auto table_pair = [&](int j, int64_t* pb) {  // -2: behind the prefix
        for (int b = 0; b < 2; ++b) {
            const int blk = 2 * j + b;
            pb[b] = blk * kBlockTokens < p.prefix_len ? phys_block(v, p.prefix_seq, blk) : -2;
        }
    };
    int issued = pc.done;
    int64_t next_pb[2];
    table_pair(pc.j0, next_pb);
    for (int i = 0; i < pc.nk; ++i) {
        const int n = pc.done + i, st = n % kShStages;
        const int64_t pb[2] = {next_pb[0], next_pb[1]};
        if (i + 1 < pc.nk) table_pair(pc.j0 + i + 1, next_pb);
        if (n >= kShStages && !sh_wait(p, sm, &empties[st], ((n / kShStages) - 1) & 1)) break;
        int64_t rows[2];
        uint32_t bytes = 0;
        for (int b = 0; b < 2; ++b) {
            rows[b] = -1;
            if (pb[b] == -2) continue;
            if (pb[b] < 0) {
                record_status(p.status, HX_ERR_CAPACITY);
                continue;
            }
            rows[b] = (pb[b] * v.block_stride + (int64_t)pc.h * v.head_stride) / 256;
            bytes += kShRegion;
        }
        mbar_arrive_expect_tx(&fulls[st], bytes);
        uint8_t(*dst)[kShRegion] = sm.ring[is_k ? st : kShStages + st];
        const CUtensorMap* tm = is_k ? tm_k : tm_v;
        const int64_t row0 = is_k ? v.k_row0 : v.v_row0;
        for (int b = 0; b < 2; ++b) {
            if (rows[b] < 0) continue;
            const int r = (int)(row0 + rows[b]), off = b * (kShRegion / 2);
            tma_load_2d(dst[0] + off, tm, 0, r, &fulls[st], pol);
            tma_load_2d(dst[1] + off, tm, 64, r, &fulls[st], pol);
        }
        issued = n + 1;
    }
    // copies in flight land before the ring changes hands (bounded)
    if (is_k) mbar_wait(&sm.q_full, pc.index & 1);
    for (int n = max(pc.done, issued - kShStages); n < issued; ++n)
        mbar_wait(&fulls[n % kShStages], (n / kShStages) & 1);
}

// One warp, of which a lane issues.  S_0, S_1, then per tile PV_j in two key halves and S_{j+2}; S_j
// in TMEM columns 128 (j & 1), O_w (key half w) in 256 + 128 w; P_j lies over
// its own half's S columns.
__device__ void prefix_mma(const SharedParams& p, SharedSmem& sm, const PrefixPiece& pc, uint32_t tmem)
{
    const uint32_t id_qk = umma_idesc(false), id_pv = umma_idesc(true);
    const uint64_t q_desc = umma_desc(smem_u32(sm.q[0]), 16, 1024);
    const uint64_t k_desc = umma_desc(smem_u32(sm.ring[0][0]), 16, 1024);
    const uint64_t v_desc = umma_desc(smem_u32(sm.ring[kShStages][0]), kShRegion, 1024);
    constexpr uint64_t kStageStep = (2 * kShRegion) >> 4;
    auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, sh_wait(p, sm, bar, parity)) != 0; };
    bool ok = wait(&sm.q_full, pc.index & 1);
    auto issue_s = [&](int n) {
        const int ks = n % kShStages;
        if (!wait(&sm.k_full[ks], (n / kShStages) & 1)) return false;
        tc_fence_after();
        const uint64_t kd = k_desc + (uint64_t)ks * kStageStep;
        if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < 8; ++kk) {
                const uint64_t off = (uint64_t)(((kk >> 2) * kShRegion + (kk & 3) * 32) >> 4);
                umma_f16(tmem + 128 * (n & 1), q_desc + off, kd + off, id_qk, kk > 0);
            }
            umma_commit(&sm.s_full[n & 1]);
            umma_commit(&sm.k_empty[ks]);
        }
        return true;
    };
    const int n0 = pc.done, n1 = pc.done + pc.nk;
    if (ok) ok = issue_s(n0);
    if (ok && n0 + 1 < n1) ok = issue_s(n0 + 1);
    for (int n = n0; ok && n < n1; ++n) {
        const int vs = n % kShStages;
        if (!wait(&sm.v_full[vs], (n / kShStages) & 1)) break;
        for (int w = 0; w < 2 && ok; ++w) {
            if (!wait(&sm.p_full[w][n & 1], (n >> 1) & 1)) {
                ok = false;
                break;
            }
            tc_fence_after();
            const uint64_t vd = v_desc + (uint64_t)vs * kStageStep;
            if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                    umma_f16_ts(tmem + 256 + 128 * w, tmem + 128 * (n & 1) + 64 * w + 8 * kk,
                                vd + (uint64_t)(((4 * w + kk) * 2048) >> 4), id_pv, (n > n0 || kk > 0) ? 1u : 0u);
                umma_commit(&sm.pv_done[w][n & 1]);
            }
        }
        if (!ok) break;
        if (elect_one()) umma_commit(&sm.v_empty[vs]);
        if (n + 2 < n1) ok = issue_s(n + 2);
    }
    if (elect_one()) umma_commit(&sm.mma_idle);  // every MMA has finished before the piece ends
    if (!mbar_wait(&sm.mma_idle, pc.index & 1)) {
        record_status(p.status, HX_ERR_TIMEOUT);
        atomicExch(&sm.abort_flag, 1);
    }
}

// Warpgroup wg takes key columns 64 wg .. 64 wg + 63 of every tile with its own
// running max, sum and accumulator, thread t (mod 128) query row t.  A warp
// whose 32 rows are all behind the last sequence only keeps the barriers
// going: its P is whatever TMEM holds, which reaches its own rows of O alone.
__device__ void prefix_softmax(const SharedParams& p, SharedSmem& sm, const PrefixPiece& pc, uint32_t tmem, int warp,
                               int lane)
{
    const int t = threadIdx.x & 127, wg = threadIdx.x >> 7;
    const int rows = p.group * min(p.seqs_per_tile, p.n_seqs - pc.rt * p.seqs_per_tile);
    const bool live = 32 * (warp & 3) < rows;
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t o_col = 256 + 128 * wg;
    const float sc = p.scale_log2;
    float m_run = -INFINITY, l = 0.f;  // (scaled, log2 domain)
    bool ok = true;
    for (int i = 0; i < pc.nk; ++i) {
        const int n = pc.done + i, b = n & 1;
        // tcgen05.ld/st are warp-collective: every branch around them is warp-uniform
        if (!__all_sync(0xffffffffu, sh_wait(p, sm, &sm.s_full[b], (n >> 1) & 1))) {
            ok = false;
            break;
        }
        const int k0 = kShKeys * (pc.j0 + i) + 64 * wg;
        const int lim = p.prefix_len - k0;  // keys c < lim of this half exist
        if (live) {
            tc_fence_after();
            float sv[64];
            tmem_ld32(lane_base + 128 * b + 64 * wg, sv);
            tmem_ld32(lane_base + 128 * b + 64 * wg + 32, sv + 32);
            tmem_ld_wait();
            if (lim < 64) {
#pragma unroll
                for (int c = 0; c < 64; ++c) sv[c] = c < lim ? sv[c] : -INFINITY;
            }
            float mx8[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) mx8[e] = sv[e];
#pragma unroll
            for (int c = 8; c < 64; c += 8)
#pragma unroll
                for (int e = 0; e < 8; ++e) mx8[e] = fmaxf(mx8[e], sv[c + e]);
#pragma unroll
            for (int w = 4; w; w >>= 1)
#pragma unroll
                for (int e = 0; e < w; ++e) mx8[e] = fmaxf(mx8[e], mx8[e + w]);
            const float mt = mx8[0] * sc;  // the scale is positive
            // the reference max moves only when it grew by more than 2^8; the
            // whole warp then rescales its O rows, the others by exactly 1
            const bool grow = mt > m_run + 8.f;
            const float alpha = grow ? fast_exp2(m_run - mt) : 1.f;
            if (i >= 1 && __any_sync(0xffffffffu, alpha < 1.f)) {
                if (!__all_sync(0xffffffffu, sh_wait(p, sm, &sm.pv_done[wg][(n - 1) & 1], ((n - 1) >> 1) & 1))) {
                    ok = false;
                    break;
                }
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float ov[32];
                    tmem_ld32(lane_base + o_col + 32 * c, ov);
                    tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 32; ++e) ov[e] *= alpha;
                    tmem_st32(lane_base + o_col + 32 * c, ov);
                }
                tmem_st_wait();
            }
            if (grow) {
                l *= alpha;
                m_run = mt;
            }
            // P in fp16, the type of V and of the MMA: off by half a step, 2^-11
            // of a weight, or 2^-25 of the reference's for those below 2^-14 of it
            const float nm = m_run == -INFINITY ? 0.f : -m_run;
            uint32_t pw[32];
            float l8[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < 32; ++c) {
                const float p0 = fast_exp2(fmaf(sv[2 * c], sc, nm));
                const float p1 = fast_exp2(fmaf(sv[2 * c + 1], sc, nm));
                l8[c & 7] += p0 + p1;
                pw[c] = pack_half2(p0, p1);
            }
            l += ((l8[0] + l8[1]) + (l8[2] + l8[3])) + ((l8[4] + l8[5]) + (l8[6] + l8[7]));
            tmem_st32u(lane_base + 128 * b + 64 * wg, pw);
            tmem_st_wait();
        }
        if (lim < 64) {
            // V rows behind the prefix hold stale bytes: zero this half's, so
            // that 0 * garbage cannot reach O (two threads per key row)
            const int vs = n % kShStages;
            if (!__all_sync(0xffffffffu, sh_wait(p, sm, &sm.v_full[vs], (n / kShStages) & 1))) {
                ok = false;
                break;
            }
            const int key = t & 63, dh = t >> 6;
            if (key >= lim) {
#pragma unroll
                for (int ch = 0; ch < 8; ++ch)
                    *reinterpret_cast<uint4*>(sm.ring[kShStages + vs][dh] + (64 * wg + key) * 128 + ch * 16) =
                        make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[wg][b]);
    }
    const int last = pc.done + pc.nk - 1;
    const bool have_o = __all_sync(0xffffffffu, ok && sh_wait(p, sm, &sm.pv_done[0][last & 1], (last >> 1) & 1) &&
                                                    sh_wait(p, sm, &sm.pv_done[1][last & 1], (last >> 1) & 1));
    // The halves' (m, l) go through the idle K ring; each warpgroup combines
    // O_0 and O_1 for its half of the dims and stores them row beside row.
    float2* ml = reinterpret_cast<float2*>(&sm.ring[0][0][0]);  // [2][128]
    ml[wg * 128 + t] = make_float2(m_run, l);
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (have_o && live) {
        tc_fence_after();
        const float2 ml0 = ml[t], ml1 = ml[128 + t];
        const float m = fmaxf(ml0.x, ml1.x);
        const float a0 = ml0.x == -INFINITY ? 0.f : fast_exp2(ml0.x - m);
        const float a1 = ml1.x == -INFINITY ? 0.f : fast_exp2(ml1.x - m);
        float o0[64], o1[64];
        tmem_ld32(lane_base + 256 + 64 * wg, o0);
        tmem_ld32(lane_base + 256 + 64 * wg + 32, o0 + 32);
        tmem_ld32(lane_base + 384 + 64 * wg, o1);
        tmem_ld32(lane_base + 384 + 64 * wg + 32, o1 + 32);
        tmem_ld_wait();
        if (t < rows) {
            float4* dst = reinterpret_cast<float4*>(p.pre_o) + (pc.slot * 32 + 16 * wg) * 128 + t;
#pragma unroll
            for (int e = 0; e < 16; ++e)
                dst[e * 128] = make_float4(o0[4 * e] * a0 + o1[4 * e] * a1, o0[4 * e + 1] * a0 + o1[4 * e + 1] * a1,
                                           o0[4 * e + 2] * a0 + o1[4 * e + 2] * a1,
                                           o0[4 * e + 3] * a0 + o1[4 * e + 3] * a1);
            if (wg == 0) p.pre_ml[pc.slot * 128 + t] = make_float2(m, a0 * ml0.y + a1 * ml1.y);
        }
    }
    fence_proxy_async_smem();  // the next copies into the K ring come after these accesses
    tc_fence_before();
}

// ------------------------------------------------------------------ suffix

// The copies of a warp's suffix steps, K and V in turn, into its ring.  The
// table's entries come in windows of 32 blocks of one sequence, one a lane.
struct SuffixFeed {
    SuffixCursor at;
    int next, total;          // halves (K or V of a step) issued, and to issue
    int seq, first;           // the window: blocks [first, first + 32) of seq
    int64_t pb;               // this lane's entry
    int64_t rel;              // rows from the layer's base to the step's, or -1

    // Starts the next half; the whole warp calls it.
    __device__ void issue(const SharedParams& p, const CUtensorMap* tm_k, const CUtensorMap* tm_v, uint8_t* ring,
                          uint64_t* full, uint64_t pol, int lane)
    {
        if (next >= total) return;
        const KVView& v = p.view;
        const bool is_v = next & 1;
        if (!is_v) {
            const int pos0 = (p.prefix_len / kShSufKeys + at.j) * kShSufKeys, blk = pos0 / kBlockTokens;
            if (at.seq != seq || blk < first || blk >= first + 32) {
                seq = at.seq;
                first = blk;
                pb = phys_block(v, seq, blk + lane);
            }
            const int64_t b = __shfl_sync(0xffffffffu, pb, blk - first);
            rel = b < 0 ? -1 : (b * v.block_stride + (int64_t)at.h * v.head_stride) / 256 + pos0 % kBlockTokens;
        }
        const int slot = next % kShSufRing;
        if (lane == 0) {
            if (rel < 0) {
                record_status(p.status, HX_ERR_CAPACITY);  // no copy: the row's result is void
                mbar_arrive(&full[slot]);
            } else {
                const int row = (int)((is_v ? v.v_row0 : v.k_row0) + rel);
                uint8_t* dst = ring + slot * kShSufSlot;
                mbar_arrive_expect_tx(&full[slot], kShSufSlot);
                tma_load_2d(dst, is_v ? tm_v : tm_k, 0, row, &full[slot], pol);
                tma_load_2d(dst + kShSufBox, is_v ? tm_v : tm_k, 64, row, &full[slot], pol);
            }
        }
        if (is_v) at.next(p);
        ++next;
    }
};

// One warp's suffix steps [first, first + count): S^T = K Q^T (keys are M, the
// segment's rows N, in NT tiles of 8), O^T += V^T P^T.
template <int NT>
__device__ void suffix_warp(const SharedParams& p, SharedSmem& sm, const CUtensorMap* tm_k, const CUtensorMap* tm_v,
                            const SeqSteps& seqs, int64_t first, int count, int number, int warp, int lane)
{
    const int g = lane >> 2, t4 = lane & 3;
    const int lm_mi = lane >> 3, lm_r = lane & 7;
    const int64_t n_seg = (int64_t)p.n_seqs * p.view.hkv * p.chunks;
    uint8_t* ring = &sm.ring[0][0][0] + warp * kShSufRing * kShSufSlot;
    uint64_t* full = sm.suf_full[warp];
    if (lane == 0) {
        for (int i = 0; i < kShSufRing; ++i) mbar_init(&full[i], 1);
        fence_mbar_init();
    }
    __syncwarp();
    const uint64_t pol = l2_evict_first_policy();
    SuffixCursor cur = seqs.find(p, lane, first);
    SuffixFeed feed{cur, 0, 2 * count, -1, 0, -1, -1};
    for (int i = 0; i < kShSufRing; ++i) feed.issue(p, tm_k, tm_v, ring, full, pol, lane);
    // a half's arrival; false once a wait ran out (the copies behind it then
    // land first, bounded, and the warp gives up)
    auto arrived = [&](int half) {
        if (__all_sync(0xffffffffu, mbar_wait(&full[half % kShSufRing], (uint32_t)(half / kShSufRing) & 1))) return true;
        if (lane == 0) {
            record_status(p.status, HX_ERR_TIMEOUT);
            for (int k = half + 1; k < feed.next; ++k)
                mbar_wait(&full[k % kShSufRing], (uint32_t)(k / kShSufRing) & 1);
        }
        return false;
    };
    // up to 8 rows: q in registers; up to 16: in the warp's part of the idle Q
    // buffer (16-byte chunk ch of row r at ch ^ (r & 7))
    uint32_t qb[NT == 1 ? 8 : 1][2];
    uint8_t* qs = sm.q[0] + warp * 16 * 256;
    float o[NT][8][4];             // dims 16 mt + g (+ 8) x rows 8 nt + 2 t4 (+ 1)
    float m[NT][2], l[NT][2];      // rows 8 nt + 2 t4 + c: reference max (log2 domain), this lane's sum
    int64_t slot = 0;
    for (int i = 0; i < count; ++i) {
        if (i == 0 || cur.j == 0) {
            slot = cur.j == 0 ? cur.segment(p) : n_seg + number;
            const int rows = min(p.chunk, p.group - cur.rc * p.chunk);
            const __half* q = p.q + ((int64_t)cur.s * p.hq + cur.h * p.group + cur.rc * p.chunk) * 128;
            if constexpr (NT == 1) {
#pragma unroll
                for (int kk = 0; kk < 8; ++kk)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        qb[kk][e] = g < rows ? *reinterpret_cast<const uint32_t*>(q + g * 128 + 16 * kk + 2 * t4 + 8 * e)
                                             : 0u;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int r = 2 * e + (lane >> 4), ch = lane & 15;
                    *reinterpret_cast<uint4*>(qs + r * 256 + ((ch ^ (r & 7)) << 4)) =
                        r < rows ? *reinterpret_cast<const uint4*>(q + r * 128 + 8 * ch) : make_uint4(0, 0, 0, 0);
                }
                __syncwarp();
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int mt = 0; mt < 8; ++mt) o[nt][mt][0] = o[nt][mt][1] = o[nt][mt][2] = o[nt][mt][3] = 0.f;
                m[nt][0] = m[nt][1] = -INFINITY;
                l[nt][0] = l[nt][1] = 0.f;
            }
        }
        if (!arrived(2 * i)) return;
        const uint32_t kb = smem_u32(ring + 2 * i % kShSufRing * kShSufSlot);
        const int key = 8 * (lm_mi >> 1) + lm_r;
        // S of the step's two 16-key tiles; independent accumulators for the
        // even and odd dims of one n-tile, or for two n-tiles
        constexpr int kChains = NT == 1 ? 2 : 1;
        float sc[2][kChains][NT][4];
#pragma unroll
        for (int c = 0; c < 2 * kChains * NT * 4; ++c) (&sc[0][0][0][0])[c] = 0.f;
#pragma unroll(8 / NT)
        for (int kk = 0; kk < 8; ++kk) {
            const int ch = 2 * kk + (lm_mi & 1);
            uint32_t b0, b1, b2, b3;
            if constexpr (NT == 1) {
                b0 = qb[kk][0];
                b1 = qb[kk][1];
            } else {  // rows 0-7: dims 16 kk .., + 8; rows 8-15 likewise
                ldmatrix_x4(b0, b1, b2, b3, smem_u32(qs) + key * 256 + ((ch ^ lm_r) << 4));
            }
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                uint32_t r0, r1, r2, r3;
                ldmatrix_x4(r0, r1, r2, r3, kb + (ch >> 3) * kShSufBox + (16 * kt + key) * 128 + (((ch & 7) ^ lm_r) << 4));
                const uint32_t a[4] = {r0, r2, r1, r3};
                mma_16816(sc[kt][kk % kChains][0], a, b0, b1);
                if constexpr (NT == 2) mma_16816(sc[kt][0][1], a, b2, b3);
            }
        }
        __syncwarp();  // K has been read
        feed.issue(p, tm_k, tm_v, ring, full, pol, lane);
        const int pos0 = (p.prefix_len / kShSufKeys + cur.j) * kShSufKeys;
        const int lo = p.prefix_len - pos0, hi = cur.len - pos0;  // own keys of the step: [lo, hi)
        const bool edge = lo > 0 || hi < kShSufKeys;
        uint32_t pb[2][NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            // x[kt][e]: key 16 kt + g + 8 (e / 2), row 8 nt + 2 t4 + (e % 2)
            float x[2][4];
            bool grow = false;
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float sum = kChains == 2 ? sc[kt][0][nt][e] + sc[kt][kChains - 1][nt][e] : sc[kt][0][nt][e];
                    const int at = 16 * kt + g + 8 * (e >> 1);
                    x[kt][e] = edge && (at < lo || at >= hi) ? -INFINITY : sum * p.scale_log2;
                    // the reference moves only when a score passes it by 2^8, so
                    // that a step without one needs no maximum over the lanes
                    grow |= x[kt][e] > m[nt][e & 1] + 8.f;
                }
            if (__any_sync(0xffffffffu, grow)) {
                float al[2];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float mx = fmaxf(fmaxf(x[0][c], x[0][c + 2]), fmaxf(x[1][c], x[1][c + 2]));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                    const float mn = fmaxf(m[nt][c], mx);
                    al[c] = mn == -INFINITY ? 1.f : fast_exp2(m[nt][c] - mn);
                    m[nt][c] = mn;
                    l[nt][c] *= al[c];
                }
#pragma unroll
                for (int mt = 0; mt < 8; ++mt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[nt][mt][e] *= al[e & 1];
            }
            float ref[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) ref[c] = m[nt][c] == -INFINITY ? 0.f : m[nt][c];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                float pr[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) pr[e] = fast_exp2(x[kt][e] - ref[e & 1]);
                l[nt][0] += pr[0] + pr[2];
                l[nt][1] += pr[1] + pr[3];
                // P^T in fp16, as V is (off as in the prefix)
                pb[kt][nt][0] = movmatrix_trans(pack_half2(pr[0], pr[1]));
                pb[kt][nt][1] = movmatrix_trans(pack_half2(pr[2], pr[3]));
            }
        }
        if (!arrived(2 * i + 1)) return;
        uint8_t* vs = ring + (2 * i + 1) % kShSufRing * kShSufSlot;
        if (edge) {
            // V rows outside hold other or stale bytes: 0 * garbage must not reach O
            for (int c = lane; c < kShSufKeys * 16; c += 32) {
                const int row = c >> 4, ch = c & 15;
                if (row < lo || row >= hi)
                    *reinterpret_cast<uint4*>(vs + (ch >> 3) * kShSufBox + row * 128 + (ch & 7) * 16) =
                        make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
            __syncwarp();
        }
        const uint32_t vb = smem_u32(vs);
#pragma unroll
        for (int mt = 0; mt < 8; ++mt) {
            const int ch = 2 * mt + (lm_mi & 1);
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                uint32_t a[4];
                ldmatrix_x4_trans(a[0], a[1], a[2], a[3],
                                  vb + (ch >> 3) * kShSufBox + (16 * kt + key) * 128 + (((ch & 7) ^ lm_r) << 4));
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_16816(o[nt][mt], a, pb[kt][nt][0], pb[kt][nt][1]);
            }
        }
        __syncwarp();  // V has been read
        feed.issue(p, tm_k, tm_v, ring, full, pol, lane);
        if (cur.j == cur.steps - 1 || i == count - 1) {
            const int rows = min(p.chunk, p.group - cur.rc * p.chunk);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float sum = l[nt][c];
                    sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                    const int r = 8 * nt + 2 * t4 + c;
                    if (r >= rows) continue;
                    float* dst = p.suf_o + (slot * p.chunk + r) * 128 + g;
#pragma unroll
                    for (int mt = 0; mt < 8; ++mt) {
                        dst[16 * mt] = o[nt][mt][c];
                        dst[16 * mt + 8] = o[nt][mt][c + 2];
                    }
                    if (g == 0) p.suf_ml[slot * p.chunk + r] = make_float2(m[nt][c], sum);
                }
        }
        cur.next(p);
    }
}

// ------------------------------------------------------------------ the launch

template <int NT>
__global__ void __launch_bounds__(kShThreads, 1)
    shared_decode_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                         const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm32_k,
                         const __grid_constant__ CUtensorMap tm32_v, const SharedParams p)
{
    extern __shared__ uint8_t smem_raw[];
    auto& sm = *reinterpret_cast<SharedSmem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cta = blockIdx.x;
    // What needs no input comes first.  Whether the CTA has prefix tiles is not
    // known yet; TMEM is taken all the same, by one warp beside the others' planning.
    if (threadIdx.x == 0) {
        prefetch_tensormap(&tm_q);
        prefetch_tensormap(&tm_k);
        prefetch_tensormap(&tm_v);
        mbar_init(&sm.q_full, 1);
        for (int i = 0; i < kShStages; ++i) {
            mbar_init(&sm.k_full[i], 1);
            mbar_init(&sm.k_empty[i], 1);
            mbar_init(&sm.v_full[i], 1);
            mbar_init(&sm.v_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sm.s_full[i], 1);
            for (int w = 0; w < 2; ++w) {
                mbar_init(&sm.p_full[w][i], 4);
                mbar_init(&sm.pv_done[w][i], 1);
            }
        }
        mbar_init(&sm.mma_idle, 1);
        sm.abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == kShMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                         smem_u32(&sm.tmem_base))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pdl_wait();  // inputs come from the previous kernel on the stream
    pdl_trigger();  // only now: the combine reads them before its own wait
    {
        // every warp plans for itself: a suffix warp waits for no other
        const SeqSteps seqs(p, lane, cta == 0 && warp == 0);
        const SharedPlan plan(p, seqs.total(p, lane, 0, nullptr, cta == 0 && warp == 0), lane);
        if (cta >= plan.pre) {
            if (warp == kShMmaWarp) {
                __syncwarp();
                asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(
                                 *reinterpret_cast<volatile uint32_t*>(&sm.tmem_base))
                             : "memory");
            }
            const int number = warp * (p.ctas - plan.pre) + cta - plan.pre;
            if (warp >= kShSoftmaxWarps || number >= plan.suf) return;
            const int64_t first = split_first(plan.n_suf, plan.suf, number);
            const int count = (int)(split_first(plan.n_suf, plan.suf, number + 1) - first);
            suffix_warp<NT>(p, sm, &tm32_k, &tm32_v, seqs, first, count, number, warp, lane);
            return;
        }
        if (threadIdx.x == 0) {
            sm.pre0 = split_first(plan.n_pre, plan.pre, cta);
            sm.pre1 = split_first(plan.n_pre, plan.pre, cta + 1);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem_base;
    PrefixPiece pc{};
    for (int64_t t = sm.pre0; t < sm.pre1;) {
        const int64_t seg = t / p.key_tiles;  // kv head * row tiles + row tile
        pc.h = (int)(seg / p.row_tiles);
        pc.rt = (int)(seg % p.row_tiles);
        pc.j0 = (int)(t % p.key_tiles);
        pc.nk = (int)min((int64_t)(p.key_tiles - pc.j0), sm.pre1 - t);
        pc.slot = pc.j0 == 0 ? seg : (int64_t)p.view.hkv * p.row_tiles + blockIdx.x;
        if (warp == kShProducerWarp) {
            if (lane < 2) prefix_producer(p, sm, pc, &tm_q, &tm_k, &tm_v, lane);
        } else if (warp == kShMmaWarp) {
            prefix_mma(p, sm, pc, tmem);
        } else {
            prefix_softmax(p, sm, pc, tmem, warp, lane);
        }
        tc_fence_before();
        __syncthreads();  // the piece's copies, MMAs and TMEM reads are done
        tc_fence_after();
        const bool stop = sm.abort_flag;
        __syncthreads();  // read by all before another wait may set it
        if (stop) break;
        t += pc.nk;
        pc.done += pc.nk;
        ++pc.index;
    }
    __syncthreads();
    if (warp == kShMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// Merges the pieces: a CTA takes eight consecutive rows of a row tile, 16
// threads a row (dims 4 i .. and 4 (i + 16) ..), the slices of threads every
// SLICES-th piece.  Rows lie beside each other in a prefix slot, so a warp's
// loads are 128-byte runs.  Bound by the chain of its dependent loads: four
// slices let two CTAs share an SM, so that those of a wide call are resident
// at once; eight shorten the chain when few row tiles have many pieces each.
constexpr int kShCombineRows = 8;

template <int SLICES>
__global__ void __launch_bounds__(128 * SLICES, 8 / SLICES)
    shared_combine_kernel(const SharedParams p, int row_chunks)
{
    pdl_trigger();
    const int tid = threadIdx.x & 127, slice = threadIdx.x >> 7, lane = threadIdx.x & 31;
    const int row8 = blockIdx.x % row_chunks;
    const int rt = blockIdx.x / row_chunks % p.row_tiles, h = blockIdx.x / row_chunks / p.row_tiles;
    const int r = row8 * kShCombineRows + tid % kShCombineRows, c = tid / kShCombineRows;
    const int s = rt * p.seqs_per_tile + r / p.group, gq = r % p.group;
    const bool row = r < p.seqs_per_tile * p.group && s < p.n_seqs;
    // Before the wait, while the main kernel's last CTAs run: all that the
    // inputs say (every CTA there has seen them complete, and none writes them).
    const SeqSteps seqs(p, lane, false);
    int64_t before = 0;
    const SharedPlan plan(p, seqs.total(p, lane, row ? s : 0, &before, false), lane);
    const int len = row ? row_length(p, s, false) : -1;
    const int64_t pre_segs = (int64_t)p.view.hkv * p.row_tiles, suf_segs = (int64_t)p.n_seqs * p.view.hkv * p.chunks;
    int64_t pre_seg = 0, suf_seg = 0;
    int pre_c = 0, pre_n = 0, suf_c = 0, suf_n = 0;  // first part that holds the segment, and how many do
    if (len > 0 && p.key_tiles > 0) {
        pre_seg = (int64_t)h * p.row_tiles + rt;
        pre_c = split_owner(plan.n_pre, plan.pre, pre_seg * p.key_tiles);
        pre_n = split_owner(plan.n_pre, plan.pre, (pre_seg + 1) * p.key_tiles - 1) - pre_c + 1;
    }
    const int steps = len > 0 ? suffix_steps(p, len) : 0;
    const int rc = gq / p.chunk, rr = gq % p.chunk;
    if (steps > 0) {
        suf_seg = ((int64_t)s * p.view.hkv + h) * p.chunks + rc;
        const int64_t t0 = before * p.view.hkv * p.chunks + (int64_t)(h * p.chunks + rc) * steps;
        suf_c = split_owner(plan.n_suf, plan.suf, t0);
        suf_n = split_owner(plan.n_suf, plan.suf, t0 + steps - 1) - suf_c + 1;
    }
    pdl_wait();  // the pieces come from the main kernel
    float M = -INFINITY, L = 0.f;
    float4 acc[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
    auto add = [&](float2 ml, float4 a, float4 b) {
        const float Mn = fmaxf(M, ml.x);
        const float Mu = Mn == -INFINITY ? 0.f : Mn;
        const float x = fast_exp2(M - Mu), y = fast_exp2(ml.x - Mu);
        L = L * x + ml.y * y;
        acc[0].x = acc[0].x * x + a.x * y; acc[0].y = acc[0].y * x + a.y * y;
        acc[0].z = acc[0].z * x + a.z * y; acc[0].w = acc[0].w * x + a.w * y;
        acc[1].x = acc[1].x * x + b.x * y; acc[1].y = acc[1].y * x + b.y * y;
        acc[1].z = acc[1].z * x + b.z * y; acc[1].w = acc[1].w * x + b.w * y;
        M = Mn;
    };
    // Pieces 0 .. pre_n - 1 are the prefix's, the rest the suffix's; a slice's
    // loads of two pieces are in flight together.
    for (int i0 = slice; i0 < pre_n + suf_n; i0 += 2 * SLICES) {
        float2 ml[2];
        float4 a[2], b[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int i = i0 + u * SLICES, k = i - pre_n;
            ml[u] = make_float2(-INFINITY, 0.f);
            a[u] = b[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (i < pre_n) {
                const int64_t slot = i == 0 ? pre_seg : pre_segs + pre_c + i;
                const float4* o = reinterpret_cast<const float4*>(p.pre_o) + slot * 32 * 128 + r;
                ml[u] = __ldcg(&p.pre_ml[slot * 128 + r]);
                a[u] = __ldcg(o + c * 128);
                b[u] = __ldcg(o + (c + 16) * 128);
            } else if (k < suf_n) {
                const int64_t slot = k == 0 ? suf_seg : suf_segs + suf_c + k;
                const float4* o = reinterpret_cast<const float4*>(p.suf_o) + (slot * p.chunk + rr) * 32;
                ml[u] = __ldcg(&p.suf_ml[slot * p.chunk + rr]);
                a[u] = __ldcg(o + c);
                b[u] = __ldcg(o + c + 16);
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) add(ml[u], a[u], b[u]);
    }
    __shared__ float2 sh_ml[SLICES][kShCombineRows];
    __shared__ float4 sh_acc[SLICES][2][128];
    if (c == 0) sh_ml[slice][tid % kShCombineRows] = make_float2(M, L);
    sh_acc[slice][0][tid] = acc[0];
    sh_acc[slice][1][tid] = acc[1];
    __syncthreads();
    if (slice > 1 || len < 0) return;  // slices 0 and 1 store the lower and upper dims
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (len > 0) {
        M = -INFINITY;
        for (int i = 0; i < SLICES; ++i) M = fmaxf(M, sh_ml[i][tid % kShCombineRows].x);
        const float Mu = M == -INFINITY ? 0.f : M;
        L = 0.f;
        for (int i = 0; i < SLICES; ++i) {
            const float2 ml = sh_ml[i][tid % kShCombineRows];
            const float y = fast_exp2(ml.x - Mu);
            const float4 a = sh_acc[i][slice][tid];
            L += ml.y * y;
            v.x += a.x * y; v.y += a.y * y; v.z += a.z * y; v.w += a.w * y;
        }
        v = make_float4(v.x / L, v.y / L, v.z / L, v.w / L);
    }
    const int64_t at = ((int64_t)s * p.hq + h * p.group + gq) * 128 + 4 * (c + 16 * slice);
    if (p.out_f32) *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = v;
    else *reinterpret_cast<uint2*>(static_cast<__half*>(p.out) + at) = make_uint2(pack_half2(v.x, v.y), pack_half2(v.z, v.w));
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

// The tensor-core path takes head_dim 128 and groups that fit a row tile.
static bool shared_fast(const hx_kv_cache* c, int group)
{
    return c->has_tmap && c->cfg.head_dim == 128 && group <= kShRows;
}

// Fills in the shape-dependent fields of the fast path.
static void shared_shape(const hx_kv_cache* c, SharedParams& p)
{
    p.seqs_per_tile = kShRows / p.group;
    p.row_tiles = (p.n_seqs + p.seqs_per_tile - 1) / p.seqs_per_tile;
    p.chunk = std::min(p.group, 16);
    p.chunks = (p.group + p.chunk - 1) / p.chunk;
    p.key_tiles = (p.prefix_len + kShKeys - 1) / kShKeys;
    p.ctas = num_sms();
}

// Workspace: pre_o, pre_ml, suf_o, suf_ml.  Returns its bytes, and
// binds it to p when ws is given.
static size_t shared_workspace(const SharedParams& shape, int hkv, void* ws, SharedParams* p)
{
    const size_t pre = (size_t)hkv * shape.row_tiles + shape.ctas;
    const size_t suf = ((size_t)shape.n_seqs * hkv * shape.chunks + shape.ctas * kShSoftmaxWarps) * shape.chunk;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        char* ptr = static_cast<char*>(ws) + at;
        at += (bytes + 15) / 16 * 16;
        return ptr;
    };
    void* a = take(pre * kShRows * 128 * sizeof(float));
    void* b = take(pre * kShRows * sizeof(float2));
    void* d = take(suf * 128 * sizeof(float));
    void* e = take(suf * sizeof(float2));
    if (p) {
        p->pre_o = static_cast<float*>(a);
        p->pre_ml = static_cast<float2*>(b);
        p->suf_o = static_cast<float*>(d);
        p->suf_ml = static_cast<float2*>(e);
    }
    return at;
}

static size_t shared_ws_bytes(const hx_kv_cache* c, int n_seqs, int num_q_heads, int prefix_len)
{
    SharedParams p{};
    p.n_seqs = n_seqs;
    p.group = num_q_heads / c->cfg.num_kv_heads;
    p.prefix_len = prefix_len;
    if (!shared_fast(c, p.group)) return 16;
    shared_shape(c, p);
    return shared_workspace(p, c->cfg.num_kv_heads, nullptr, nullptr);
}

template <int NT>
static int launch_shared(const hx_kv_cache* c, const SharedParams& p, const CUtensorMap& tm_q, cudaStream_t s)
{
    auto kernel = shared_decode_kernel<NT>;
    const size_t smem = sizeof(SharedSmem) + 1024;
    static std::atomic<bool> attr_set[64];  // per device; set again on ordinals past 63
    int dev = 0;
    HX_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !attr_set[dev].load(std::memory_order_acquire)) {
        HX_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        if (dev >= 0 && dev < 64) attr_set[dev].store(true, std::memory_order_release);
    }
    cudaError_t e = launch_kernel(kernel, dim3(p.ctas), dim3(kShThreads), smem, s, true, tm_q, c->tm_k, c->tm_v,
                                  c->tm32_k, c->tm32_v, p);
    if (e != cudaSuccess) return cuda_fail(e, "shared_decode_kernel launch");
    if (int rc = check_launch("shared_decode_kernel")) return rc;
    const int row_chunks = (std::min(p.n_seqs, p.seqs_per_tile) * p.group + kShCombineRows - 1) / kShCombineRows;
    const int64_t segments = (int64_t)p.view.hkv * p.row_tiles;
    const dim3 grid((unsigned)(segments * row_chunks));
    const bool wide = p.ctas > 16 * segments;
    e = wide ? launch_kernel(shared_combine_kernel<8>, grid, dim3(1024), 0, s, true, p, row_chunks)
             : launch_kernel(shared_combine_kernel<4>, grid, dim3(512), 0, s, true, p, row_chunks);
    if (e != cudaSuccess) return cuda_fail(e, "shared_combine_kernel launch");
    return check_launch("shared_combine_kernel");
}

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
    if (!shared_fast(c, p.group)) {
        shared_generic_kernel<<<n_seqs * num_q_heads, 128, 0, (cudaStream_t)stream>>>(p);
        return check_launch("shared_generic_kernel");
    }
    shared_shape(c, p);
    shared_workspace(p, hkv, workspace, &p);
    // q as [sequence][q head][128]: one box is a row tile's half of the dims
    CUtensorMap tm_q;
    const uint64_t dims[3] = {128, (uint64_t)num_q_heads, (uint64_t)n_seqs};
    const uint64_t strides[2] = {256, (uint64_t)num_q_heads * 256};
    const uint32_t box[3] = {64, (uint32_t)p.group, (uint32_t)p.seqs_per_tile};
    if (int rc = encode_fp16_map(&tm_q, 3, q, dims, strides, box)) return rc;
    cudaStream_t s = (cudaStream_t)stream;
    return p.chunk <= 8 ? launch_shared<1>(c, p, tm_q, s) : launch_shared<2>(c, p, tm_q, s);
}
