// Attention of the new tokens of a batch over the paged cache, on the 5th-generation
// tensor cores.
//
//   s = scale q . k,  p = exp(s - max),  o = sum p v / sum p,  lse = max + ln sum p
//
// over the slots that the token sees; o times sigmoid(gate) where a gate is given.
// A row that sees nothing gives o = 0 and lse = -inf.
//
// One pass over the cache per tile of query rows, a running maximum and sum per row.
//  - Rows: the G = H / KVH query heads of a kv head share its keys, so a tile's 128 rows
//    are floor(128 / G) tokens times G heads (row = token * G + head): a single token
//    with 8 heads per kv head reads K and V once, not 8 times.
//  - A kv step is 128 slots: S = Q K^T (128 x 128, f32, tensor memory), weights P back
//    into tensor memory over S as 16-bit pairs, O += P V with P as the MMA's A operand.
//    K tiles are K-major operands and V tiles MN-major ones straight from the page
//    layout: nothing is transposed.
//  - One thread owns a row (a tensor memory lane): maximum and sum need no shuffles.
//    The exponentials are taken against a reference that follows the maximum only when
//    it has grown by more than 2^8, so O is rarely rescaled; P <= 2^8 keeps its relative
//    precision, and f32 sums divide the reference out at the end.
//  - P is rounded to the cache's type (the tensor core wants A and B alike): a relative
//    error of 2^-11 (f16) or 2^-8 (bf16) a weight, of the size of the output's own
//    rounding.  Its sum is taken before that rounding.
//  - NQ = 2: two row tiles share each K and V tile, a softmax warpgroup each (head sizes
//    up to 128).  NQ = 1: one row tile and one softmax warpgroup, two S buffers so
//    that the next scores are computed meanwhile (256-wide heads, whose O takes
//    half of tensor memory, and calls of up to 128 rows a kv head).
//  - Two threads issue MMAs, each for its own S buffer (units of one parity): a thread
//    that waits or commits holds up its own MMAs only.
//
// Work split.  The kv steps of all (sequence, kv head, row tile) items lie on one line,
// and each CTA takes an equal stretch of it, found on the device from the batch's
// lengths: ragged batches, causal chunks and single long sequences all give every SM
// the same number of steps.  An item that a stretch boundary cuts leaves partial (O,
// max, sum) in the workspace; the CTA that finishes last merges them, in the order of
// the stretches, so the result does not depend on which one that is.
//
// Warp roles: softmax warpgroups first (a warp reaches the tensor memory lanes of its
// number modulo 4), then TMA, the two MMA warps (which also clear the V rows past a
// sequence's length: 0 * NaN is NaN, and those slots may hold anything), and a warp that
// walks the work line for the others.
#include <algorithm>

#include "launch.cuh"
#include "tc_f16.cuh"

namespace w4a8 {

namespace {

constexpr int kTile = 128;                  // rows of a query tile, and slots of a kv step
constexpr uint32_t kChunkBytes = kTile * 128;  // 128 rows x 64 elements
constexpr int kSegs = 4;
constexpr int kMaxStages = 12;
constexpr uint32_t kMiscBytes = 2048;
constexpr float kLazy = 8.0f;  // log2 of how far the maximum may pass its reference

struct AttnParams {
    int H, KVH, D, G;
    int tpt;       // tokens of a row tile
    float scale;
    const float* gate;
    int gate_row, gate_head;
    void* o;
    int o_type;
    float* lse;
    int max_q, max_kv;
    int box_rows;  // slots of a TMA box
    CacheOrder order;
    int rows_cap;  // rows of a partial
    uint32_t* counters;  // [CTA][NQ]
    float* part;         // [CTA][2][NQ][rows_cap][D]
    float2* ml;          // [CTA][2][NQ][rows_cap]
    unsigned int* err;
    PagedCache c;
    PagedBatch b;
};

// A stretch of one item's kv steps.
struct Segment {
    int seq, kh;
    int tok, n;    // first new token of the tile (global row), and how many it has (up to NQ * tpt)
    int vis;       // last slot its first token sees
    int len;
    int j0, j1;    // kv steps; j1 == 0: the line's end
    int first, parts;  // first CTA of the item, CTAs that share it
};

template <int NCH, int NQ>
struct Plan {
    static constexpr int kCps = NCH == 4 ? 2 : NCH;  // 64-wide chunks of a ring stage
    static constexpr int kParts = NCH / kCps;        // stages of a K or V tile
    static constexpr uint32_t kStageBytes = kCps * kChunkBytes;
    static constexpr uint32_t kQBytes = NQ * NCH * kChunkBytes;
    static constexpr int kFit = static_cast<int>((227 * 1024 - 1024 - kMiscBytes - kQBytes) / kStageBytes);
    static constexpr int kStages = kFit < kMaxStages ? kFit : kMaxStages;
    static constexpr size_t kSmem = 1024 + kQBytes + kStages * kStageBytes + kMiscBytes;
    static constexpr int kSoftWarps = 4 * NQ;
    static constexpr int kThreads = (kSoftWarps + 4) * 32;
    static_assert(kStages >= 2 * kParts + (kParts == 1 ? 1 : 0), "ring too short");
};

struct Bars {
    uint64_t full[kMaxStages], empty[kMaxStages];
    uint64_t s_full[2], p_full[2], o_done[2];
    uint64_t q_full, q_empty;
    uint64_t seg_full[kSegs], seg_empty[kSegs];
    uint64_t group[2];
    Segment seg[kSegs];
    uint32_t last[2];
    uint32_t tmem;
    int abort;
};
static_assert(sizeof(Bars) <= kMiscBytes, "barriers exceed their space");

__device__ __forceinline__ int kv_steps(int vis_last, int len) {
    const int end = min(max(vis_last + 1, 0), len);
    return max((end + kTile - 1) / kTile, 1);  // a tile that sees nothing still writes its zeros
}

// The batch as the work line sees it: new tokens and slots within the call's bounds.
__device__ __forceinline__ SeqSpan line_span(const AttnParams& p, int seq) {
    return seq_span(p.b, p.c, seq);
}

// kv steps of one kv head of a sequence.
__device__ __forceinline__ int seq_steps(const SeqSpan& s, int n, int tpc) {
    int total = 0;
    for (int i = 0; i < n; i += tpc) total += kv_steps(s.len - s.n + min(i + tpc, n) - 1, s.len);
    return total;
}

template <typename T, int NCH, int NQ>
__global__ void __launch_bounds__(Plan<NCH, NQ>::kThreads, 1)
    attn_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                   const __grid_constant__ CUtensorMap tm_v, const AttnParams p) {
    using P = Plan<NCH, NQ>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* ring = smem + P::kQBytes;
    Bars& bars = *reinterpret_cast<Bars*>(ring + P::kStages * P::kStageBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kTmaWarp = P::kSoftWarps, kMmaWarp = kTmaWarp + 1, kLineWarp = kTmaWarp + 3;

    if (threadIdx.x == 0) {
        for (int s = 0; s < P::kStages; ++s) {
            mbar_init(&bars.full[s], 1);
            mbar_init(&bars.empty[s], 2);  // both MMA warps, whether they use the tile or not
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars.s_full[i], 1);
            mbar_init(&bars.p_full[i], 4);
            mbar_init(&bars.o_done[i], 1);
            mbar_init(&bars.group[i], 128);
        }
        mbar_init(&bars.q_full, 1);
        mbar_init(&bars.q_empty, 2);
        for (int i = 0; i < kSegs; ++i) {
            mbar_init(&bars.seg_full[i], 1);
            mbar_init(&bars.seg_empty[i], P::kSoftWarps + 3);
        }
        bars.abort = 0;
        mbar_init_fence();
    }
    if (warp == kMmaWarp) tmem1_alloc(&bars.tmem, 512);
    tc1_fence_before();
    __syncthreads();
    tc1_fence_after();
    const uint32_t tmem = bars.tmem;
    constexpr uint32_t kO = 256;  // first column of O (of the first row tile)
    pdl_launch_dependents();
    pdl_wait();

    const Bail bail{&bars.abort, p.err};
    const int tpc = NQ * p.tpt;  // tokens of an item
    // The next segment, for every role but the line's; false at the end.
    uint32_t sq = 0;
    auto next_seg = [&](Segment& s) -> bool {
        const uint32_t i = sq % kSegs;
        const bool ok = !*bail.flag && bail.wait(&bars.seg_full[i], (sq / kSegs) & 1);
        if (!__all_sync(kFull, ok)) return false;
        s = bars.seg[i];
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.seg_empty[i]);
        ++sq;
        return s.j1 > 0;
    };

    if (warp == kLineWarp) {
        // ---- the work line: this CTA's stretch of it, segment by segment ----
        long long total = 0;
        for (int b0 = 0; b0 < p.b.batch; b0 += 32) {
            long long mine = 0;
            if (b0 + lane < p.b.batch) {
                const SeqSpan s = line_span(p, b0 + lane);
                mine = static_cast<long long>(seq_steps(s, min(s.n, p.max_q), tpc)) * p.KVH;
            }
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) mine += __shfl_xor_sync(kFull, mine, off);
            total += mine;
        }
        const long long ctas = min(static_cast<long long>(gridDim.x), total);
        const long long c = blockIdx.x;
        long long at = 0, end = 0;
        if (c < ctas) {
            at = c * total / ctas;
            end = (c + 1) * total / ctas;
        }
        // the CTA whose stretch holds step x
        auto cta_of = [&](long long x) { return static_cast<int>(((x + 1) * ctas - 1) / total); };
        uint32_t sk = 0;
        bool ok = true;
        auto publish = [&](const Segment& s) -> bool {
            const uint32_t i = sk % kSegs;
            ok = ok && !*bail.flag && bail.wait(&bars.seg_empty[i], ((sk / kSegs) & 1) ^ 1);
            if (!__all_sync(kFull, ok)) return ok = false;
            if (lane == 0) {
                bars.seg[i] = s;
                mbar_arrive(&bars.seg_full[i]);
            }
            ++sk;
            return true;
        };
        // the sequence that holds step `at`, and the line position of its start
        int seq = 0;
        long long base = 0;
        if (at < end) {
            for (int b0 = 0; b0 < p.b.batch; b0 += 32) {
                long long mine = 0;
                if (b0 + lane < p.b.batch) {
                    const SeqSpan s = line_span(p, b0 + lane);
                    mine = static_cast<long long>(seq_steps(s, min(s.n, p.max_q), tpc)) * p.KVH;
                }
                long long upto = mine;
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) {
                    const long long y = __shfl_up_sync(kFull, upto, off);
                    if (lane >= off) upto += y;
                }
                const unsigned past = __ballot_sync(kFull, base + upto > at);
                if (past) {
                    const int f = __ffs(past) - 1;
                    seq = b0 + f;
                    base += __shfl_sync(kFull, upto - mine, f);
                    break;
                }
                base += __shfl_sync(kFull, upto, 31);
            }
        }
        SeqSpan s{};
        int n = 0, kh = 0, i = 0, steps = 0;  // item: kv head kh, tokens from i
        long long item = base;                // its position
        if (at < end) {
            s = line_span(p, seq);
            n = min(s.n, p.max_q);
            const long long per = seq_steps(s, n, tpc);
            kh = static_cast<int>((at - base) / per);
            item = base + kh * per;
            for (;; i += tpc) {
                steps = kv_steps(s.len - s.n + min(i + tpc, n) - 1, s.len);
                if (item + steps > at) break;
                item += steps;
            }
        }
        while (at < end && ok) {
            Segment g;
            g.seq = seq;
            g.kh = kh;
            g.tok = s.t0 + i;
            g.n = min(tpc, n - i);
            g.vis = s.len - s.n + i;
            g.len = s.len;
            g.j0 = static_cast<int>(at - item);
            g.j1 = static_cast<int>(min(static_cast<long long>(steps), end - item));
            g.first = cta_of(item);
            g.parts = cta_of(item + steps - 1) - g.first + 1;
            if (!publish(g)) break;
            at += g.j1 - g.j0;
            item += steps;
            i += tpc;
            if (i >= n) {
                i = 0;
                if (++kh == p.KVH) {
                    kh = 0;
                    do {
                        if (++seq >= p.b.batch) break;
                        s = line_span(p, seq);
                        n = min(s.n, p.max_q);
                    } while (n == 0);
                }
            }
            if (at < end) steps = kv_steps(s.len - s.n + min(i + tpc, n) - 1, s.len);
        }
        Segment stop{};
        if (ok) publish(stop);
    } else if (warp == kTmaWarp) {
        // ---- TMA: the tiles in the order in which the MMAs use them ----
        //  NQ = 1: K0 K1 V0 K2 V1 ...   NQ = 2: K0 V0 K1 V1 ...
        // (the last V of the line keeps its place, one past a K that is not there)
        uint32_t pos_max = 0;
        bool ok = true;
        uint32_t u = 0, qs = 0;  // kv steps so far, query loads so far
        const int boxes = kTile / p.box_rows;
        const uint32_t box_bytes = static_cast<uint32_t>(p.box_rows) * 128;
        // page and row of this lane's box of step j
        auto locate = [&](const Segment& g, int j, int& page, int& row, int& n) {
            const int s0 = j * kTile + lane * p.box_rows;
            n = min(boxes, max((g.len - j * kTile + p.box_rows - 1) / p.box_rows, 0));
            page = 0;
            row = 0;
            if (lane < n) {
                const int pi = s0 / p.c.page;
                page = static_cast<int>(page_of(p.b, p.c, g.seq, pi));
                row = s0 - pi * p.c.page;
            }
        };
        auto load = [&](const CUtensorMap* map, uint32_t pos, int kh, int page, int row, int n) -> bool {
            for (int part = 0; part < P::kParts; ++part) {
                const uint32_t st = (pos + part) % P::kStages;
                ok = ok && !*bail.flag && bail.wait(&bars.empty[st], (((pos + part) / P::kStages) & 1) ^ 1);
                if (!__all_sync(kFull, ok)) return ok = false;
                if (lane == 0) {
                    if (n > 0)
                        mbar_expect_tx(&bars.full[st], static_cast<uint32_t>(n) * box_bytes * P::kCps);
                    else
                        mbar_arrive(&bars.full[st]);
                }
                __syncwarp();
                if (lane < n) {
                    const uint32_t dst = smem_u32(ring + st * P::kStageBytes) + lane * box_bytes;
#pragma unroll
                    for (int ch = 0; ch < P::kCps; ++ch)
                        tma_load_4d(dst + ch * kChunkBytes, map, (part * P::kCps + ch) * 64, p.order.pick(0, row, kh, page),
                                    p.order.pick(1, row, kh, page), p.order.pick(2, row, kh, page), &bars.full[st]);
                }
                pos_max = max(pos_max, pos + part + 1);
            }
            return true;
        };
        Segment g;
        int vpage = 0, vrow = 0, vn = 0, vkh = 0;  // the V tile still to come (NQ = 1)
        while (ok && next_seg(g)) {
            ok = ok && !*bail.flag && bail.wait(&bars.q_empty, (qs & 1) ^ 1);
            if (!__all_sync(kFull, ok)) {
                ok = false;
                break;
            }
            if (lane == 0) {
                const uint32_t bytes = static_cast<uint32_t>(p.tpt) * p.G * 128;
                mbar_expect_tx(&bars.q_full, bytes * NCH * NQ);
                for (int t = 0; t < NQ; ++t)
                    for (int ch = 0; ch < NCH; ++ch)
                        tma_load_3d_at(smem_u32(smem + (t * NCH + ch) * kChunkBytes), &tm_q, ch * 64, g.kh * p.G,
                                       g.tok + t * p.tpt, &bars.q_full);
            }
            ++qs;
            for (int j = g.j0; j < g.j1 && ok; ++j, ++u) {
                int page, row, n;
                locate(g, j, page, row, n);
                if (NQ == 2) {
                    if (load(&tm_k, 2 * u * P::kParts, g.kh, page, row, n)) load(&tm_v, (2 * u + 1) * P::kParts, g.kh, page, row, n);
                } else {
                    if (load(&tm_k, (u == 0 ? 0 : 2 * u - 1) * P::kParts, g.kh, page, row, n) && u > 0)
                        load(&tm_v, 2 * u * P::kParts, vkh, vpage, vrow, vn);
                    vpage = page;
                    vrow = row;
                    vn = n;
                    vkh = g.kh;
                }
            }
        }
        if (NQ == 1 && ok && u > 0) load(&tm_v, 2 * u * P::kParts, vkh, vpage, vrow, vn);
        // no copy may still be landing when the CTA exits (a place that was skipped was filled one round earlier)
        for (uint32_t s = 0; s < P::kStages; ++s) {
            // the last fill of this stage
            uint32_t last = 0;
            bool any = false;
            for (uint32_t q = pos_max > 2 * P::kStages ? pos_max - 2 * P::kStages : 0; q < pos_max; ++q) {
                const bool skipped = NQ == 1 && u > 0 && q >= (2 * u - 1) * P::kParts && q < 2 * u * P::kParts;
                if (q % P::kStages == s && !skipped) {
                    last = q;
                    any = true;
                }
            }
            if (any) mbar_wait(&bars.full[s], (last / P::kStages) & 1);
        }
        if (qs > 0) mbar_wait(&bars.q_full, (qs - 1) & 1);
    } else if (warp == kMmaWarp || warp == kMmaWarp + 1) {
        // ---- MMA: S(u) = Q K(u)^T once P of this buffer's previous unit has been used by O += P V ----
        const int w = warp - kMmaWarp;  // S buffer, and row tile where there are two
        constexpr uint32_t id_qk = idesc_f16<T>(kTile, false), id_pv = idesc_f16<T>(P::kCps * 64, true);
        const uint32_t s_tm = tmem + w * 128;
        const uint32_t o_tm = tmem + kO + (NQ == 2 ? w * NCH * 64 : 0);
        const uint32_t q_sm = smem_u32(smem) + (NQ == 2 ? w * NCH * kChunkBytes : 0);
        bool ok = true;
        // Both warps follow every fill of the ring in order, so a wait for a stage's phase
        // always comes after that stage's phase before (a parity wait that is a phase early
        // would return at once); a tile that is the other warp's is released unused.
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            ok = ok && !*bail.flag && bail.wait(bar, parity);
            return ok = __all_sync(kFull, ok);
        };
        auto tile_wait = [&](uint32_t pos) {
            for (int part = 0; part < P::kParts; ++part)
                if (!wait(&bars.full[(pos + part) % P::kStages], ((pos + part) / P::kStages) & 1)) return false;
            return true;
        };
        auto tile_skip = [&](uint32_t pos) {
            if (!tile_wait(pos)) return;
            if (lane == 0)
                for (int part = 0; part < P::kParts; ++part) mbar_arrive(&bars.empty[(pos + part) % P::kStages]);
            __syncwarp();
        };
        auto own = [&](uint32_t u) { return NQ == 2 || (u & 1) == static_cast<uint32_t>(w); };
        // O += P(u) V; valid < 128 where the V tile reaches past the sequence
        auto pv = [&](uint32_t u, bool first, int valid) {
            const uint32_t pos = (NQ == 2 ? 2 * u + 1 : 2 * u + 2) * P::kParts;
            if (!own(u)) return tile_skip(pos);
            if (!tile_wait(pos)) return;
            if (valid < kTile) {
                // clear the rows of slots past the length (NQ = 2: both warps, the same zeros)
                for (int part = 0; part < P::kParts; ++part) {
                    unsigned char* v = ring + ((pos + part) % P::kStages) * P::kStageBytes;
                    for (int e = valid * 8 + lane; e < kTile * 8; e += 32)
#pragma unroll
                        for (int ch = 0; ch < P::kCps; ++ch)
                            *reinterpret_cast<uint4*>(v + ch * kChunkBytes + e * 16) = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async();
                __syncwarp();
            }
            if (!wait(&bars.p_full[w], (NQ == 2 ? u : u >> 1) & 1)) return;
            // one O: the units take turns, each after the one before
            if (NQ == 1 && u > 0 && !wait(&bars.o_done[w ^ 1], ((u - 1) >> 1) & 1)) return;
            tc1_fence_after();
            if (lane == 0) {
#pragma unroll
                for (int part = 0; part < P::kParts; ++part) {
                    const uint32_t st = (pos + part) % P::kStages;
                    const uint32_t v = smem_u32(ring + st * P::kStageBytes);
#pragma unroll
                    for (int kk = 0; kk < kTile / 16; ++kk)
                        mma_f16_ts(o_tm + part * P::kCps * 64, s_tm + kk * 8, desc_mn_major(v + kk * 2048, kChunkBytes),
                                   id_pv, !first || kk > 0);
                    tc1_commit(&bars.empty[st]);
                }
                tc1_commit(&bars.o_done[w]);
            }
            __syncwarp();
        };
        // S(u) = Q K^T; fresh: the segment's Q has not been waited for
        auto qk = [&](uint32_t u, bool& fresh, uint32_t seg) {
            const uint32_t pos = (NQ == 2 ? 2 * u : (u == 0 ? 0 : 2 * u - 1)) * P::kParts;
            if (!own(u)) return tile_skip(pos);
            if (fresh && !wait(&bars.q_full, seg & 1)) return;
            fresh = false;
            for (int part = 0; part < P::kParts; ++part) {
                if (!wait(&bars.full[(pos + part) % P::kStages], ((pos + part) / P::kStages) & 1)) return;
                tc1_fence_after();
                if (lane == 0) {
                    const uint32_t st = (pos + part) % P::kStages;
                    const uint32_t k = smem_u32(ring + st * P::kStageBytes);
#pragma unroll
                    for (int ch = 0; ch < P::kCps; ++ch)
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            mma_f16_ss(s_tm, desc_k_major(q_sm + (part * P::kCps + ch) * kChunkBytes + kk * 32),
                                       desc_k_major(k + ch * kChunkBytes + kk * 32), id_qk, part + ch + kk > 0);
                    tc1_commit(&bars.empty[st]);
                }
                __syncwarp();
            }
            if (lane == 0) tc1_commit(&bars.s_full[w]);
            __syncwarp();
        };
        uint32_t u = 0, segs = 0;
        bool have = false, first = false;  // the unit before u: its P V is due
        int valid = kTile;
        Segment g;
        while (ok && next_seg(g)) {
            bool fresh = true;
            for (int j = g.j0; j < g.j1 && ok; ++j, ++u) {
                // in the ring's order: NQ = 2: V(u - 1) K(u), NQ = 1: K(u) V(u - 1)
                if (NQ == 2 && have) pv(u - 1, first, valid);
                if (ok) qk(u, fresh, segs);
                if (NQ == 1 && have && ok) pv(u - 1, first, valid);
                have = true;
                first = j == g.j0;
                valid = max(min(g.len - j * kTile, kTile), 0);
            }
            // through with the segment's Q: a warp that had no unit in it comes after its load all the same,
            // or its arrival could count for the segment before
            if (ok && fresh) wait(&bars.q_full, segs & 1);
            if (!ok) break;
            if (lane == 0) tc1_commit(&bars.q_empty);
            __syncwarp();
            ++segs;
        }
        if (ok && have) pv(u - 1, first, valid);
    } else {
        // ---- softmax, one thread a row, and the output ----
        const int grp = NQ == 2 ? warp / 4 : 0;
        const int r = (warp & 3) * 32 + lane;  // row of the tile
        const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t o_tm = tmem + lane_off + kO + grp * NCH * 64;
        const float c = p.scale * 1.44269504088896340736f;
        const int tok_in = r / p.G, head_in = r - tok_in * p.G;
        uint32_t u = 0, gphase = 0;  // units so far of this group
        bool ok = true;
        // O after unit x of this group
        auto o_wait = [&](uint32_t x) {
            ok = !*bail.flag && bail.wait(&bars.o_done[NQ == 2 ? grp : (x & 1)], (NQ == 2 ? x : x >> 1) & 1);
            ok = __all_sync(kFull, ok);
            if (ok) tc1_fence_after();
            return ok;
        };
        auto group_sync = [&]() {
            mbar_arrive(&bars.group[grp]);
            ok = bail.wait(&bars.group[grp], gphase & 1) && ok;
            ++gphase;
            return ok;
        };
        Segment g;
        while (ok && next_seg(g)) {
            const int toks = min(max(g.n - grp * p.tpt, 0), p.tpt);
            const bool live = tok_in < toks;  // (rows past tpt * G have tok_in >= tpt)
            const bool any_live = __any_sync(kFull, live);
            const int lim = live ? g.vis + grp * p.tpt + tok_in : -1;  // last slot this row sees
            int least = live ? lim : 0x7fffffff;
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) least = min(least, __shfl_xor_sync(kFull, least, off));
            float m = -INFINITY, l = 0.f;
            for (int j = g.j0; j < g.j1 && ok; ++j, ++u) {
                const uint32_t buf = NQ == 2 ? grp : (u & 1), use = NQ == 2 ? u : u >> 1;
                ok = !*bail.flag && bail.wait(&bars.s_full[buf], use & 1);
                if (!__all_sync(kFull, ok)) {
                    ok = false;
                    break;
                }
                tc1_fence_after();
                if (any_live) {
                    const uint32_t s_tm = tmem + lane_off + buf * 128;
                    float s[kTile];
#pragma unroll
                    for (int i = 0; i < kTile; i += 32) tmem1_ld32(s_tm + i, s + i);
                    tmem1_wait_ld();
                    const int kv0 = j * kTile;
                    if (kv0 + kTile - 1 > min(least, g.len - 1)) {
                        const int lm = min(lim, g.len - 1) - kv0;
#pragma unroll
                        for (int i = 0; i < kTile; ++i)
                            if (i > lm) s[i] = -INFINITY;
                    }
                    float m0 = s[0], m1 = s[1], m2 = s[2], m3 = s[3];
#pragma unroll
                    for (int i = 4; i < kTile; i += 4) {
                        m0 = fmaxf(m0, s[i]);
                        m1 = fmaxf(m1, s[i + 1]);
                        m2 = fmaxf(m2, s[i + 2]);
                        m3 = fmaxf(m3, s[i + 3]);
                    }
                    const float mx = fmaxf(fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)), m);
                    if (__any_sync(kFull, live && (mx - m) * c > kLazy)) {
                        const float f = mx == m ? 1.f : ex2((m - mx) * c);
                        m = mx;
                        l *= f;
                        if (j > g.j0) {
                            if (!o_wait(u - 1)) break;
#pragma unroll 1
                            for (int i = 0; i < NCH * 64; i += 16) {
                                float o[16];
                                tmem1_ld16(o_tm + i, o);
                                tmem1_wait_ld();
#pragma unroll
                                for (int e = 0; e < 16; ++e) o[e] *= f;
                                tmem1_st16(o_tm + i, reinterpret_cast<const uint32_t*>(o));
                            }
                        }
                    }
                    const float neg = m == -INFINITY ? 0.f : -m * c;
                    const float2 c2 = make_float2(c, c), neg2 = make_float2(neg, neg);
                    float2 l0 = make_float2(0.f, 0.f), l1 = make_float2(0.f, 0.f);
#pragma unroll
                    for (int h = 0; h < kTile; h += 64) {
                        uint32_t w[32];
#pragma unroll
                        for (int i = 0; i < 64; i += 4) {
                            float2 a = __ffma2_rn(make_float2(s[h + i], s[h + i + 1]), c2, neg2);
                            float2 b = __ffma2_rn(make_float2(s[h + i + 2], s[h + i + 3]), c2, neg2);
                            a.x = ex2(a.x);
                            a.y = ex2(a.y);
                            b.x = ex2(b.x);
                            b.y = ex2(b.y);
                            l0 = __fadd2_rn(l0, a);
                            l1 = __fadd2_rn(l1, b);
                            w[i / 2] = Elem<T>::pack(a.x, a.y);
                            w[i / 2 + 1] = Elem<T>::pack(b.x, b.y);
                        }
                        tmem1_st32(s_tm + h / 2, w);
                    }
                    l += (l0.x + l0.y) + (l1.x + l1.y);
                    tmem1_wait_st();
                    tc1_fence_before();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars.p_full[buf]);
            }
            if (!ok) break;
            if (!o_wait(u - 1)) break;
            const int h = g.kh * p.G + head_in;
            const int t = g.tok + grp * p.tpt + tok_in;
            // 16 columns of a row into the output, scaled, gated, rounded
            auto put = [&](int tt, int hh, int col, float* o, float f) {
                if (p.gate) {
                    const float4* gp = reinterpret_cast<const float4*>(p.gate + static_cast<size_t>(tt) * p.gate_row +
                                                                       static_cast<size_t>(hh) * p.gate_head + col);
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const float4 x = ld_dep(gp + e / 4);
                        o[e] *= f / (1.f + __expf(-x.x));
                        o[e + 1] *= f / (1.f + __expf(-x.y));
                        o[e + 2] *= f / (1.f + __expf(-x.z));
                        o[e + 3] *= f / (1.f + __expf(-x.w));
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] *= f;
                }
                const size_t at = (static_cast<size_t>(tt) * p.H + hh) * p.D + col;
                if (p.o_type == W4A8_F32) {
                    float4* d = reinterpret_cast<float4*>(static_cast<float*>(p.o) + at);
#pragma unroll
                    for (int e = 0; e < 16; e += 4) d[e / 4] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                } else {
                    uint4* d = reinterpret_cast<uint4*>(static_cast<T*>(p.o) + at);
#pragma unroll
                    for (int e = 0; e < 16; e += 8) {
                        uint4 x;
                        x.x = Elem<T>::pack(Elem<T>::sat(o[e]), Elem<T>::sat(o[e + 1]));
                        x.y = Elem<T>::pack(Elem<T>::sat(o[e + 2]), Elem<T>::sat(o[e + 3]));
                        x.z = Elem<T>::pack(Elem<T>::sat(o[e + 4]), Elem<T>::sat(o[e + 5]));
                        x.w = Elem<T>::pack(Elem<T>::sat(o[e + 6]), Elem<T>::sat(o[e + 7]));
                        d[e / 8] = x;
                    }
                }
            };
            if (g.parts == 1) {
                if (any_live) {
                    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
                    for (int col = 0; col < p.D; col += 16) {
                        float o[16];
                        tmem1_ld16(o_tm + col, o);
                        tmem1_wait_ld();
                        if (live) put(t, h, col, o, inv);
                        __syncwarp();
                    }
                    if (live && p.lse) p.lse[static_cast<size_t>(t) * p.H + h] = l == 0.f ? -INFINITY : m * p.scale + logf(l);
                }
                continue;
            }
            // a shared item: this CTA's part, then the merge by whoever comes last
            const int rows = toks * p.G;
            auto slot = [&](int cta) {
                return (static_cast<size_t>(cta) * 2 + (cta == g.first ? 1 : 0)) * NQ + grp;
            };
            if (any_live) {
                const size_t sl = slot(blockIdx.x);
                float* dst = p.part + (sl * p.rows_cap + r) * p.D;
#pragma unroll 1
                for (int col = 0; col < p.D; col += 16) {
                    float o[16];
                    tmem1_ld16(o_tm + col, o);
                    tmem1_wait_ld();
                    if (live) {
#pragma unroll
                        for (int e = 0; e < 16; e += 4)
                            __stcg(reinterpret_cast<float4*>(dst + col + e), make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]));
                    }
                    __syncwarp();
                }
                if (live) __stcg(p.ml + sl * p.rows_cap + r, make_float2(m, l));
            }
            tc1_fence_before();
            __threadfence();
            if (!group_sync()) break;
            const int gt = threadIdx.x & 127;
            uint32_t* counter = p.counters + static_cast<size_t>(g.first) * NQ + grp;
            if (gt == 0) {
                const uint32_t before = atomicAdd(counter, 1u);
                bars.last[grp] = before == static_cast<uint32_t>(g.parts - 1);
                if (before == static_cast<uint32_t>(g.parts - 1)) *counter = 0;
                __threadfence();
            }
            if (!group_sync()) break;
            if (!bars.last[grp]) continue;
            for (int e = gt; e < rows * (p.D / 16); e += 128) {
                const int row = e / (p.D / 16), col = (e - row * (p.D / 16)) * 16;
                float top = -INFINITY;
                for (int q = 0; q < g.parts; ++q) top = fmaxf(top, __ldcg(p.ml + slot(g.first + q) * p.rows_cap + row).x);
                float o[16], sum = 0.f;
#pragma unroll
                for (int x = 0; x < 16; ++x) o[x] = 0.f;
                for (int q = 0; q < g.parts; ++q) {
                    const size_t sl = slot(g.first + q);
                    const float2 ml = __ldcg(p.ml + sl * p.rows_cap + row);
                    const float f = ml.x == top ? 1.f : ex2((ml.x - top) * c);
                    sum += f * ml.y;
                    const float4* src = reinterpret_cast<const float4*>(p.part + (sl * p.rows_cap + row) * p.D + col);
#pragma unroll
                    for (int x = 0; x < 16; x += 4) {
                        const float4 v = __ldcg(src + x / 4);
                        o[x] += f * v.x;
                        o[x + 1] += f * v.y;
                        o[x + 2] += f * v.z;
                        o[x + 3] += f * v.w;
                    }
                }
                const int tt = g.tok + grp * p.tpt + row / p.G, hh = g.kh * p.G + row % p.G;
                put(tt, hh, col, o, sum == 0.f ? 0.f : 1.f / sum);
                if (col == 0 && p.lse)
                    p.lse[static_cast<size_t>(tt) * p.H + hh] = sum == 0.f ? -INFINITY : top * p.scale + logf(sum);
            }
        }
    }

    tc1_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc1_fence_after();
        tmem1_dealloc(tmem, 512);
    }
}

PFN_cuTensorMapEncodeTiled_v12000 map_encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    });
    return fn;
}

CUtensorMapDataType map_type(int dtype) {
    return dtype == W4A8_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

w4a8_status encode(CUtensorMap* map, int dtype, int rank, const void* base, const cuuint64_t* dims,
                   const cuuint64_t* strides, const cuuint32_t* box, const char* what) {
    const PFN_cuTensorMapEncodeTiled_v12000 enc = map_encoder();
    if (!enc) return set_error(W4A8_ECUDA, "%s: cuTensorMapEncodeTiled unavailable", what);
    const cuuint32_t elem[4] = {1, 1, 1, 1};
    const CUresult r = enc(map, map_type(dtype), static_cast<cuuint32_t>(rank), const_cast<void*>(base), dims, strides, box,
                           elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(W4A8_ECUDA, "%s: tensor map: error %d", what, static_cast<int>(r));
    return W4A8_OK;
}

}  // namespace

w4a8_status encode_cache(CUtensorMap* map, CacheOrder* order, const void* base, const PagedCache& c, int KVH, int D,
                         const char* what) {
    struct Dim {
        int id;
        cuuint64_t count, stride;
        cuuint32_t box;
    } d[3] = {{0, static_cast<cuuint64_t>(c.page), static_cast<cuuint64_t>(c.row_stride) * 2,
               static_cast<cuuint32_t>(cache_box_rows(c.page))},
              {1, static_cast<cuuint64_t>(KVH), static_cast<cuuint64_t>(c.head_stride) * 2, 1},
              {2, static_cast<cuuint64_t>(c.pages), static_cast<cuuint64_t>(c.page_stride) * 2, 1}};
    // a dimension of one has no stride of its own: it goes last
    cuuint64_t most = 16;
    for (const Dim& x : d)
        if (x.count > 1) most = std::max(most, x.stride);
    for (Dim& x : d)
        if (x.count == 1) x.stride = most;
    std::stable_sort(d, d + 3, [](const Dim& x, const Dim& y) { return x.stride < y.stride; });
    cuuint64_t dims[4] = {static_cast<cuuint64_t>(D)}, strides[3];
    cuuint32_t box[4] = {64};
    for (int i = 0; i < 3; ++i) {
        dims[i + 1] = d[i].count;
        strides[i] = d[i].stride;
        box[i + 1] = d[i].box;
        order->id[i] = d[i].id;
    }
    return encode(map, c.dtype, 4, base, dims, strides, box, what);
}

w4a8_status encode_queries(CUtensorMap* map, const void* q, int dtype, int H, int D, int row_stride, int tokens, int G,
                           int box_tokens, const char* what) {
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(H), static_cast<cuuint64_t>(tokens)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(D) * 2, static_cast<cuuint64_t>(row_stride) * 2};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(G), static_cast<cuuint32_t>(box_tokens)};
    return encode(map, dtype, 3, q, dims, strides, box, what);
}

namespace {

// How a call is laid out on the GPU, from its sizes alone.
struct Layout {
    int nch, nq, tpt, rows_cap, grid;
    size_t counters, slots, bytes;
};

Layout layout_of(int H, int KVH, int D, int batch, int max_q, int max_kv, int sms) {
    Layout x{};
    const int G = H / KVH;
    x.nch = (D + 63) / 64;
    x.tpt = kTile / G;
    // two row tiles for each K and V tile where there are rows for both and O fits beside them
    x.nq = x.nch <= 2 && static_cast<long long>(max_q) * G > kTile ? 2 : 1;
    x.rows_cap = std::min(x.tpt, std::max(max_q, 1)) * G;
    const long long tiles = (static_cast<long long>(std::max(max_q, 1)) + x.nq * x.tpt - 1) / (x.nq * x.tpt);
    const long long steps = std::max((static_cast<long long>(max_kv) + kTile - 1) / kTile, 1ll);
    const long long work = std::min(tiles * steps, 1ll << 20) * KVH * batch;
    x.grid = static_cast<int>(std::min<long long>(sms, work));
    // the same place and size whatever the call, so that calls of several sizes may share a workspace
    x.counters = (static_cast<size_t>(sms) * 2 * 4 + 255) / 256 * 256;
    x.slots = static_cast<size_t>(x.grid) * 2 * x.nq * x.rows_cap;
    x.bytes = x.counters + (x.slots * 8 + 255) / 256 * 256 + x.slots * D * 4;
    return x;
}

template <typename T, int NCH, int NQ>
w4a8_status launch_tc(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const AttnParams& p, int grid,
                      cudaStream_t st) {
    using Pl = Plan<NCH, NQ>;
    const char* what = "w4a8_attn_paged";
    static FuncAttr attr;
    const w4a8_status s = ensure_smem(attn_tc_kernel<T, NCH, NQ>, attr, Pl::kSmem, -1, what);
    if (s != W4A8_OK) return s;
    return launch_pdl(what, attn_tc_kernel<T, NCH, NQ>, dim3(grid), dim3(Pl::kThreads), Pl::kSmem, st, q, k, v, p);
}

template <typename T>
w4a8_status dispatch(int nch, int nq, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                     const AttnParams& p, int grid, cudaStream_t st) {
    if (nq == 2) return nch == 1 ? launch_tc<T, 1, 2>(q, k, v, p, grid, st) : launch_tc<T, 2, 2>(q, k, v, p, grid, st);
    switch (nch) {
        case 1: return launch_tc<T, 1, 1>(q, k, v, p, grid, st);
        case 2: return launch_tc<T, 2, 1>(q, k, v, p, grid, st);
        case 3: return launch_tc<T, 3, 1>(q, k, v, p, grid, st);
        default: return launch_tc<T, 4, 1>(q, k, v, p, grid, st);
    }
}

}  // namespace

int sm_count();  // capi.cu

}  // namespace w4a8

using namespace w4a8;

extern "C" {

W4A8_API size_t w4a8_attn_paged_workspace_bytes(int32_t tokens, int32_t H, int32_t KVH, int32_t D, int32_t batch,
                                                int32_t max_q, int32_t max_kv) {
    (void)tokens;
    if (check_heads("w4a8_attn_paged_workspace_bytes", H, KVH, D) != W4A8_OK || batch < 1 || max_q < 0 || max_kv < 0)
        return 0;
    return layout_of(H, KVH, D, batch, max_q, max_kv, sm_count()).bytes;
}

W4A8_API w4a8_status w4a8_attn_paged(const void* q, int32_t q_row_stride, int32_t H, int32_t KVH, int32_t D, float scale,
                                     const float* gate, int32_t gate_row_stride, int32_t gate_head_stride,
                                     const uint32_t* q_start, const uint32_t* kv_len, const uint32_t* table,
                                     int32_t batch, int32_t table_stride, int32_t tokens, int32_t max_q, int32_t max_kv,
                                     const void* k, const void* v, int32_t dtype, int32_t pages, int32_t page,
                                     size_t page_stride, int32_t head_stride, int32_t row_stride, void* o, int32_t o_type,
                                     float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    const char* what = "w4a8_attn_paged";
    AttnParams p{};
    p.c = PagedCache{const_cast<void*>(k), const_cast<void*>(v), dtype, pages, page, page_stride, head_stride, row_stride};
    p.b = PagedBatch{q_start, kv_len, table, batch, table_stride, tokens};
    w4a8_status st = check_heads(what, H, KVH, D);
    if (st == W4A8_OK) st = check_cache(what, p.c, KVH, D);
    if (st == W4A8_OK) st = check_batch(what, p.b);
    if (st != W4A8_OK) return st;
    if (static_cast<long long>(table_stride) * page >= (1ll << 31))
        return set_error(W4A8_EINVAL, "%s: %d pages of %d slots a sequence", what, table_stride, page);
    if (tokens > 0 && (!q || !o)) return set_error(W4A8_EINVAL, "%s: NULL pointer", what);
    if (!aligned(q, 16) || !aligned(o, 16)) return set_error(W4A8_EINVAL, "%s: q and o must be 16-byte aligned", what);
    if (q_row_stride % 8 || q_row_stride < static_cast<long long>(H) * D)
        return set_error(W4A8_EINVAL, "%s: q row stride %d (a multiple of 8 that holds the heads)", what, q_row_stride);
    if (o_type != W4A8_F32 && o_type != dtype)
        return set_error(W4A8_EINVAL, "%s: output type %d (the cache's, or W4A8_F32)", what, o_type);
    if (gate && (!aligned(gate, 16) || gate_row_stride % 4 || gate_head_stride % 4 || gate_head_stride < 0 || gate_row_stride < 0))
        return set_error(W4A8_EINVAL, "%s: gate not 16-byte aligned, or strides %d, %d (multiples of 4)", what,
                         gate_row_stride, gate_head_stride);
    if (max_q < 0 || max_q > (1 << 24) || max_kv < 0)
        return set_error(W4A8_EINVAL, "%s: max_q=%d max_kv=%d", what, max_q, max_kv);
    if (!(scale > 0.f) || scale > 1e30f) return set_error(W4A8_EINVAL, "%s: scale %g", what, scale);
    const Layout x = layout_of(H, KVH, D, batch, max_q, max_kv, sm_count());
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < x.bytes)
        return set_error(W4A8_EINVAL, "%s: workspace NULL, misaligned or under %zu bytes", what, x.bytes);
    if (tokens == 0 || max_q == 0) return W4A8_OK;
    p.H = H;
    p.KVH = KVH;
    p.D = D;
    p.G = H / KVH;
    p.tpt = x.tpt;
    p.scale = scale;
    p.gate = gate;
    p.gate_row = gate_row_stride;
    p.gate_head = gate_head_stride;
    p.o = o;
    p.o_type = o_type;
    p.lse = lse;
    p.max_q = max_q;
    p.max_kv = max_kv;
    p.box_rows = cache_box_rows(page);
    p.rows_cap = x.rows_cap;
    p.counters = static_cast<uint32_t*>(workspace);
    p.ml = reinterpret_cast<float2*>(static_cast<char*>(workspace) + x.counters);
    p.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + x.counters + (x.slots * 8 + 255) / 256 * 256);
    p.err = device_error_word();
    CUtensorMap mq, mk, mv;
    st = encode_queries(&mq, q, dtype, H, D, q_row_stride, tokens, p.G, x.tpt, what);
    if (st == W4A8_OK) st = encode_cache(&mk, &p.order, k, p.c, KVH, D, what);
    if (st == W4A8_OK) st = encode_cache(&mv, &p.order, v, p.c, KVH, D, what);
    if (st != W4A8_OK) return st;
    cudaStream_t cs = static_cast<cudaStream_t>(stream);
    return dtype == W4A8_F16 ? dispatch<__half>(x.nch, x.nq, mq, mk, mv, p, x.grid, cs)
                             : dispatch<__nv_bfloat16>(x.nch, x.nq, mq, mk, mv, p, x.grid, cs);
}

}  // extern "C"
