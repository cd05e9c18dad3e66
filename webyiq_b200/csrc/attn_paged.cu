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
//  - A thread takes 64 scores of one row (a tensor memory lane) at a time: maximum and sum
//    need no shuffles.  The exponentials are taken against a reference that follows the maximum only when
//    it has grown by more than 2^8, so O is rarely rescaled, and f32 sums divide the
//    reference out at the end.
//  - P is rounded to the cache's type (the tensor core wants A and B alike): a relative
//    error of 2^-11 (f16) or 2^-8 (bf16) a weight, of the size of the output's own
//    rounding.  Its sum is taken before that rounding.  f16 weights are made 2^7 times as
//    large, so that they fill its range up to 2^15: below 2^-21 of the row's largest weight
//    they are subnormal, with an error of up to 2^-32 of it, N 2^-32 for N slots.  (Without
//    the factor 2^-25: a cache beside one slot that takes most of the weight lost its part of
//    the output where its scores lie 17 below.)  bf16 has f32's exponents.
//  - NQ = 2: two row tiles share each K and V tile, a softmax warpgroup each (head sizes up to
//    128).  A tile's S is two halves of 64 slots, so that one's scores are computed while
//    the other's weights are made, and the two tiles' warps take turns at the
//    exponentials.  NQ = 1: one row tile, two S buffers of 128 slots, and two softmax
//    warpgroups that split a row's scores and exchange their maxima through shared memory
//    (wider heads, whose O takes half of tensor memory, and calls of up to 128 rows a kv
//    head).  PAIR: two such CTAs share each K and V tile, half of it in the shared memory of
//    each (cta_group::2), for heads past 192 with more than one row tile.
//  - Two threads issue MMAs, each for its own S buffers: a thread that waits or commits
//    holds up its own MMAs only.
//
// What bounds it, measured: 2048 tokens over 16384 slots, 32 / 8 heads of 128: 446 to 480 us
// in short runs, at best 1157 TFLOP/s (0.69 of the measured bf16 burst rate), 521 to 534 back to
// back at the 1000 W limit.
// Not one unit but the hand-overs between them: a warp's 64 exponentials take 512 clocks at
// the unit's rate (611 with their sums and rounding), its half step about 1900, and S is ready in 99
// of 100 half steps; heads of 64, with two thirds of the MMAs, still take 412 us.  An MMA
// warp's delay counts, too: its waits read the abort flag only where a barrier is not
// complete.  (Whole steps of 128: 530 us, before these two steps, the scores and the
// exponentials in turn.  Two warpgroups a tile: 628.  A quarter or half of the
// exponentials by polynomial on the FMA pipe: 529, 543 where 504 stood.  The order of
// multiplies, exponentials, sums and roundings: no change.)  256-wide heads: 2048 tokens over 16384
// slots, 8 / 2 heads, in 247 us as pairs, 1044 TFLOP/s, and 276 as single CTAs, which read
// 128 KB from L2 a step of 2048 clocks; a 4001-token prompt 90 against 100, gated 113
// against 117; now 87 to 91 and 107 to 109.  Heads of 129 to 192 take single CTAs whatever the
// rows (96 KB a step of 1536 clocks): 1024 tokens over 8192 slots, 32 / 8 heads of 192, in 181 us,
// 1068 TFLOP/s, nearer the burst rate than 256-wide pairs (262 us, 983) and 128-wide double tiles
// (138 us, 932).  Heads of 80 and 96 cost nearly what 128 do (131 and 134 us).
// Single tokens: 48 sequences, 888 MB, at 5.9 TB/s in short runs (0.91 of the measured copy
// rate), 5.0 to 5.3 back to back; one token over 100003 slots 47 to 50 us, 16 to 18 above its
// bytes' time: the line, the first loads and the merge.
//
// Work split.  The kv steps of all (sequence, kv head, row tile) items lie on one line,
// and each CTA takes an equal stretch of it, found on the device from the batch's
// lengths: ragged batches, causal chunks and single long sequences all give every SM
// the same number of steps.  An item that a stretch boundary cuts leaves partial (O,
// max, sum) in the workspace, and a second, small kernel merges those, in the order of
// the stretches (by the CTA that finishes last it took 28 us for one token over 10000
// slots: one SM's threads, where the merge kernel has all of them).
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
// After how many of a half step's 64 weights the other row tile's warp may begin its own: the hand-over takes about as
// long as the rest.  2048 tokens over 16384 slots, 64-wide heads: 415, 413, 413, 419 and 414 us with 16, 32, 48, 56 and
// 64; 455 where the arrival does not depend on the weights, which the assembler then puts before them.
constexpr int kPass = 48;
constexpr uint32_t kMiscBytes = 3072;
// An item's start and end (query load, epilogue), in kv steps; a gate's loads lengthen its end.  Measured on 4001
// tokens of 8 / 2 heads of 256: 152, 127, 119, 120 and 122 us with 2, 3, 4, 6 and 8 and a gate, 102, 101, 103, 104
// and 107 without one; 48 single tokens 157, 151, 150, 151, 153.
constexpr int kItemCost = 3, kGatedItemCost = 5;
constexpr int kHalf = kTile / 2;  // scores of a row that one thread takes
constexpr float kLazy = 8.0f;  // log2 of how far the maximum may pass its reference
// log2 of the factor on a row's weights, in P, its sum and O alike: f16's largest power of two is 2^15.
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 15.0f - kLazy : 0.0f;
// A row's lse from its reference and its sum, which carries the factor (a power of two: exact).
template <typename T>
__device__ __forceinline__ float lse_of(float top, float scale, float sum) {
    constexpr float kDrop = std::is_same<T, __half>::value ? 1.0f / 128.0f : 1.0f;
    static_assert(kDrop * (1 << static_cast<int>(kLift<T>)) == 1.0f, "the factor and its inverse");
    return sum == 0.f ? -INFINITY : top * scale + logf(sum * kDrop);
}

struct AttnParams {
    int H, KVH, D, G;
    int tpt;       // tokens of a row tile
    float scale;
    const float* gate;
    int gate_row, gate_head;
    void* o;
    int o_type;
    float* lse;
    int max_q;
    int item_cost;   // kItemCost or kGatedItemCost
    int box_rows;    // slots of a TMA box
    int box_tokens;  // tokens of one
    CacheOrder order;
    int rows_cap;  // rows of a partial
    int4* shared_items;  // [CTA] the item that starts in its stretch and goes on in the next
    float4* part;        // [CTA][2][NQ][D / 4][rows_cap]
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

template <int NCH, int NQ, bool PAIR>
struct Plan {
    static constexpr int kCps = PAIR || NCH < 4 ? NCH : 2;  // 64-wide chunks of a ring stage
    static constexpr int kParts = NCH / kCps;               // stages of a K or V tile
    // a pair's CTA holds half of each tile: 64 slots of K, half the columns of V
    static constexpr uint32_t kKChunk = PAIR ? kChunkBytes / 2 : kChunkBytes;
    static constexpr int kVCps = PAIR ? NCH / 2 : kCps;
    static constexpr uint32_t kStageBytes = kCps * kKChunk;
    static constexpr int kTiles = PAIR ? 2 : NQ;  // row tiles of an item
    static_assert(!PAIR || (NQ == 1 && NCH == 4), "pairs are for one row tile a CTA and the widest heads");
    static constexpr uint32_t kQBytes = NQ * NCH * kChunkBytes;
    static constexpr int kFit = static_cast<int>((227 * 1024 - kMiscBytes - kQBytes) / kStageBytes);
    static constexpr int kStages = kFit < kMaxStages ? kFit : kMaxStages;
    static constexpr size_t kSmem = kQBytes + kStages * kStageBytes + kMiscBytes;
    static constexpr int kSoftWarps = 8;
    static constexpr int kThreads = (kSoftWarps + 4) * 32;
    static_assert(kStages + 2 * NQ < 32, "a lane each for the last waits");
    static_assert(kStages >= 2 * kParts + (kParts == 1 ? 1 : 0), "ring too short");
};

struct Bars {
    uint64_t full[kMaxStages], empty[kMaxStages];
    uint64_t s_full[2][2], p_full[2][2], o_done[2][2];  // [row tile][parity of the unit]
    uint64_t q_full, q_empty;
    uint64_t peer_full[kMaxStages], peer_q;  // the pair's other CTA has its half (in CTA 0)
    uint64_t seg_full[kSegs], seg_empty[kSegs];
    uint64_t pair[4];     // [quarter]: the two warps that share its rows (NQ = 1)
    uint64_t turn[2][4];  // [row tile][quarter]: its exponentials' turn (NQ = 2)
    Segment seg[kSegs];
    float xch[2][2][kTile];  // [turn][half][row]
    uint32_t tmem;
    int abort;
};
static_assert(sizeof(Bars) <= kMiscBytes, "barriers exceed their space");

// An arrival that waits for a value: nothing else keeps one behind arithmetic that it does not use.
__device__ __forceinline__ void arrive_after(uint64_t* bar, uint32_t value) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %1, 0xffffffff;\n @p mbarrier.arrive.shared::cta.b64 _, [%0];\n"
        " @!p mbarrier.arrive.shared::cta.b64 _, [%0];\n}\n" ::"r"(smem_u32(bar)),
        "r"(value)
        : "memory");
}

__device__ __forceinline__ int kv_steps(int vis_last, int len) {
    return (max(min(vis_last + 1, len), 1) - 1) / kTile + 1;  // a tile that sees nothing still writes its zeros
}

// Length on the work line of one kv head of this lane's sequence (n tokens, 0 for none); a warp's call.
// A sequence of many row tiles is summed by the whole warp.
__device__ __forceinline__ long long seq_length(const SeqSpan& s, int n, int tpc, int cost, int lane) {
    long long total = 0;
    const bool many = n > 4 * tpc;
    if (!many)
        for (int i = 0; i < n; i += tpc) total += kv_steps(s.len - s.n + min(i + tpc, n) - 1, s.len) + cost;
    for (unsigned todo = __ballot_sync(kFull, many); todo; todo &= todo - 1) {
        const int src = __ffs(todo) - 1;
        const int n1 = __shfl_sync(kFull, n, src), len = __shfl_sync(kFull, s.len, src), sn = __shfl_sync(kFull, s.n, src);
        long long sum = 0;
        for (int i = lane * tpc; i < n1; i += 32 * tpc) sum += kv_steps(len - sn + min(i + tpc, n1) - 1, len) + cost;
        sum = line_sum(sum);
        if (lane == src) total = sum;
    }
    return total;
}

__device__ __forceinline__ void load_gate8(const AttnParams& p, int t, int h, int col, float4* g) {
    const float4* at = reinterpret_cast<const float4*>(p.gate + static_cast<size_t>(t) * p.gate_row +
                                                       static_cast<size_t>(h) * p.gate_head + col);
    g[0] = ld_dep(at);
    g[1] = ld_dep(at + 1);
}
// Eight columns of a row into the output: scaled, gated, rounded.
template <typename T>
__device__ __forceinline__ void put8(const AttnParams& p, int t, int h, int col, float* o, float f, const float4* gate) {
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] *= f;
    if (p.gate) {
        const float* g = reinterpret_cast<const float*>(gate);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = __fdividef(o[e], 1.f + __expf(-g[e]));
    }
    const size_t at = (static_cast<size_t>(t) * p.H + h) * p.D + col;
    if (p.o_type == W4A8_F32) {
        float4* d = reinterpret_cast<float4*>(static_cast<float*>(p.o) + at);
        d[0] = make_float4(o[0], o[1], o[2], o[3]);
        d[1] = make_float4(o[4], o[5], o[6], o[7]);
    } else {
        uint4 x;
        x.x = Elem<T>::pack(Elem<T>::sat(o[0]), Elem<T>::sat(o[1]));
        x.y = Elem<T>::pack(Elem<T>::sat(o[2]), Elem<T>::sat(o[3]));
        x.z = Elem<T>::pack(Elem<T>::sat(o[4]), Elem<T>::sat(o[5]));
        x.w = Elem<T>::pack(Elem<T>::sat(o[6]), Elem<T>::sat(o[7]));
        *reinterpret_cast<uint4*>(static_cast<T*>(p.o) + at) = x;
    }
}

// Where a CTA keeps its part of an item: the item that starts in its stretch in the
// second place, the one that came over from the stretch before in the first.
template <int NQ>
__device__ __forceinline__ size_t part_slot(int cta, int first, int grp) {
    return (static_cast<size_t>(cta) * 2 + (cta == first ? 1 : 0)) * NQ + grp;
}

// The merge of shared items.  Block (x, y): the item that starts in CTA x / NQ, row tile
// x % NQ; the block's threads take 8 columns of a row each, split PG ways over the
// item's parts.  Few rows (decode) have many parts and little else to go round, many
// rows few parts.
constexpr int kMergeThreads = 256;
template <typename T, int NQ, int PG>
__global__ void __launch_bounds__(kMergeThreads) attn_merge_kernel(const AttnParams p) {
    constexpr int kE = kMergeThreads / PG;
    __shared__ float red[PG > 1 ? kMergeThreads * 10 : 1];
    pdl_launch_dependents();
    pdl_wait();
    const int first = blockIdx.x / NQ, grp = blockIdx.x % NQ;
    const int4 item = ld_dep(p.shared_items + first);
    const int parts = item.w;
    if (parts == 0) return;
    const int rows = min(max(item.y - grp * p.tpt, 0), p.tpt) * p.G;
    const int e = blockIdx.y * kE + threadIdx.x % kE, pg = threadIdx.x / kE;
    const int col8 = e / p.rows_cap, row = e - col8 * p.rows_cap;
    const bool live = col8 < p.D / 8 && row < rows;
    const float c = p.scale * 1.44269504088896340736f;
    float top = -INFINITY, sum = 0.f, o[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) o[x] = 0.f;
    if (live) {
        const size_t item_stride = static_cast<size_t>(p.D / 4) * p.rows_cap;
        constexpr int kAhead = 4;
        for (int q0 = pg; q0 < parts; q0 += PG * kAhead) {
            float2 ml[kAhead];
            float4 a[kAhead], b[kAhead];
#pragma unroll
            for (int x = 0; x < kAhead; ++x) {
                const int q = q0 + x * PG;
                ml[x] = make_float2(-INFINITY, 0.f);
                a[x] = b[x] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (q < parts) {
                    const size_t sl = part_slot<NQ>(first + q, first, grp);
                    const float4* src = p.part + sl * item_stride + static_cast<size_t>(col8) * 2 * p.rows_cap + row;
                    ml[x] = ld_dep(p.ml + sl * p.rows_cap + row);
                    a[x] = ld_dep(src);
                    b[x] = ld_dep(src + p.rows_cap);
                }
            }
            float next = top;
#pragma unroll
            for (int x = 0; x < kAhead; ++x) next = fmaxf(next, ml[x].x);
            const float keep = next == top ? 1.f : ex2((top - next) * c);
            top = next;
            sum *= keep;
#pragma unroll
            for (int x = 0; x < 8; ++x) o[x] *= keep;
#pragma unroll
            for (int x = 0; x < kAhead; ++x) {
                const float f = ml[x].x == top ? 1.f : ex2((ml[x].x - top) * c);
                sum += f * ml[x].y;
                o[0] += f * a[x].x;
                o[1] += f * a[x].y;
                o[2] += f * a[x].z;
                o[3] += f * a[x].w;
                o[4] += f * b[x].x;
                o[5] += f * b[x].y;
                o[6] += f * b[x].z;
                o[7] += f * b[x].w;
            }
        }
    }
    if (PG > 1) {
        // [value][thread]: the PG groups' partial results, merged by the first
        red[threadIdx.x] = top;
        red[kMergeThreads + threadIdx.x] = sum;
#pragma unroll
        for (int x = 0; x < 8; ++x) red[(2 + x) * kMergeThreads + threadIdx.x] = o[x];
        __syncthreads();
        if (pg > 0) return;
        float all = top;
#pragma unroll
        for (int q = 1; q < PG; ++q) all = fmaxf(all, red[q * kE + threadIdx.x]);
        float f = top == all ? 1.f : ex2((top - all) * c);
        sum *= f;
#pragma unroll
        for (int x = 0; x < 8; ++x) o[x] *= f;
#pragma unroll
        for (int q = 1; q < PG; ++q) {
            const int at = q * kE + threadIdx.x;
            f = red[at] == all ? 1.f : ex2((red[at] - all) * c);
            sum += f * red[kMergeThreads + at];
#pragma unroll
            for (int x = 0; x < 8; ++x) o[x] += f * red[(2 + x) * kMergeThreads + at];
        }
        top = all;
    }
    if (!live) return;
    const int t = item.x + grp * p.tpt + row / p.G, h = item.z * p.G + row % p.G;
    float4 gate[2];
    if (p.gate) load_gate8(p, t, h, col8 * 8, gate);
    put8<T>(p, t, h, col8 * 8, o, sum == 0.f ? 0.f : 1.f / sum, gate);
    if (col8 == 0 && p.lse) p.lse[static_cast<size_t>(t) * p.H + h] = lse_of<T>(top, p.scale, sum);
}

template <typename T, int NCH, int NQ, bool PAIR>
__global__ void __launch_bounds__(Plan<NCH, NQ, PAIR>::kThreads, 1)
    attn_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                   const __grid_constant__ CUtensorMap tm_v, const AttnParams p) {
    using P = Plan<NCH, NQ, PAIR>;
    // the swizzled tiles want 1024-byte alignment, which dynamic shared memory has where there is no static
    extern __shared__ __align__(1024) unsigned char smem[];
    if (smem_u32(smem) & 1023) {
        if (threadIdx.x == 0) atomicOr(p.err, DEV_ERR_ATTN_TIMEOUT);
        return;
    }
    unsigned char* ring = smem + P::kQBytes;
    Bars& bars = *reinterpret_cast<Bars*>(ring + P::kStages * P::kStageBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kTmaWarp = P::kSoftWarps, kMmaWarp = kTmaWarp + 1, kLineWarp = kTmaWarp + 3;
    // who shares the work line: CTAs, or pairs of them
    const int rank = PAIR ? static_cast<int>(pair_rank()) : 0;
    const int me = PAIR ? blockIdx.x / 2 : blockIdx.x, everyone = PAIR ? gridDim.x / 2 : gridDim.x;

    if (threadIdx.x == 0) {
        for (int s = 0; s < P::kStages; ++s) {
            mbar_init(&bars.peer_full[s], 1);
            mbar_init(&bars.full[s], 1);
            mbar_init(&bars.empty[s], 2);  // both MMA warps, whether they use the tile or not
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&bars.s_full[0][i], 1);
            mbar_init(&bars.p_full[0][i], PAIR ? 16 : NQ == 2 ? 4 : 8);
            mbar_init(&bars.o_done[0][i], 1);
            mbar_init(&bars.pair[i], 2);
            mbar_init(&bars.turn[0][i], 1);
            mbar_init(&bars.turn[1][i], 1);
        }
        mbar_init(&bars.q_full, 1);
        mbar_init(&bars.peer_q, 1);
        mbar_init(&bars.q_empty, 2);
        for (int i = 0; i < kSegs; ++i) {
            mbar_init(&bars.seg_full[i], 1);
            mbar_init(&bars.seg_empty[i], P::kSoftWarps + 3);
        }
        bars.abort = 0;
        mbar_init_fence();
    }
    if (warp == kMmaWarp) {
        if (PAIR)
            tmem2_alloc(&bars.tmem, 512);
        else
            tmem1_alloc(&bars.tmem, 512);
    }
    tc1_fence_before();
    if (PAIR) pair_sync();  // both CTAs' barriers are there
    __syncthreads();
    tc1_fence_after();
    const uint32_t tmem = bars.tmem;
    constexpr uint32_t kO = 256;  // first column of O (of the first row tile)
    pdl_launch_dependents();
    pdl_wait();

    const Bail bail{&bars.abort, p.err};
    const int tpc = P::kTiles * p.tpt;  // tokens of an item
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
        // span and length, all its kv heads, of sequence b0 + lane
        auto steps_of = [&](int b0, SeqSpan& o) {
            o = SeqSpan{};
            if (b0 + lane < p.b.batch) o = seq_span(p.b, p.c, b0 + lane);
            return line_heads(seq_length(o, min(o.n, p.max_q), tpc, p.item_cost, lane), p.KVH);
        };
        SeqSpan mine_span;
        int mine = 0;
        long long whole = 0;
        for (int b0 = 0; b0 < p.b.batch; b0 += 32) {
            const long long steps = steps_of(b0, mine_span);
            whole += line_sum(steps);
            mine = static_cast<int>(steps);  // (used where the whole fits)
        }
        const int total = line_length(whole, p.err);
        const int ctas = min(everyone, total);
        const int c = me;
        int at = 0, end = 0;
        if (c < ctas) {
            at = line_mul_div(c, total, ctas);
            end = line_mul_div(c + 1, total, ctas);
        }
        // the CTA whose stretch holds step x
        auto cta_of = [&](int x) { return line_mul_div(x + 1, ctas, total, 1); };
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
        // the sequence that holds step `at`, its span and length, and the line position of its start
        SeqSpan s{};
        int seq = 0, base = 0, length = 0;
        if (at < end) {
            for (int b0 = 0; b0 < p.b.batch; b0 += 32) {
                if (p.b.batch > 32) mine = static_cast<int>(steps_of(b0, mine_span));  // (one round: as above)
                int upto = mine;
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) {
                    const int y = __shfl_up_sync(kFull, upto, off);
                    if (lane >= off) upto += y;
                }
                const unsigned past = __ballot_sync(kFull, base + upto > at);
                if (past) {
                    const int f = __ffs(past) - 1;
                    seq = b0 + f;
                    base += __shfl_sync(kFull, upto - mine, f);
                    length = __shfl_sync(kFull, mine, f);
                    s = SeqSpan{__shfl_sync(kFull, mine_span.t0, f), __shfl_sync(kFull, mine_span.n, f),
                                __shfl_sync(kFull, mine_span.len, f)};
                    break;
                }
                base += __shfl_sync(kFull, upto, 31);
            }
        }
        int n = 0, kh = 0, i = 0, steps = 0;  // item: kv head kh, tokens from i
        int item = base;                      // its position
        if (at < end) {
            n = min(s.n, p.max_q);
            const int per = length / p.KVH;
            kh = (at - base) / per;
            item = base + kh * per;
            for (; i < n; i += 32 * tpc) {  // 32 row tiles at a time
                const int first = i + lane * tpc;
                steps = first < n ? kv_steps(s.len - s.n + min(first + tpc, n) - 1, s.len) : 0;
                const int mine = first < n ? steps + p.item_cost : 0;
                int upto = mine;
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) {
                    const int y = __shfl_up_sync(kFull, upto, off);
                    if (lane >= off) upto += y;
                }
                const unsigned past = __ballot_sync(kFull, item + upto > at);
                if (past) {
                    const int f = __ffs(past) - 1;
                    i += f * tpc;
                    item += __shfl_sync(kFull, upto - mine, f);
                    steps = __shfl_sync(kFull, steps, f);
                    break;
                }
                item += __shfl_sync(kFull, upto, 31);
            }
        }
        int4 shared_item = make_int4(0, 0, 0, 0);
        while (item < end && ok) {
            Segment g;
            g.seq = seq;
            g.kh = kh;
            g.tok = s.t0 + i;
            g.n = min(tpc, n - i);
            g.vis = s.len - s.n + i;
            g.len = s.len;
            // the item's steps come behind its fixed cost
            const int start = item + p.item_cost;
            g.j0 = max(at - start, 0);
            g.j1 = min(steps, end - start);
            g.first = cta_of(start);
            g.parts = cta_of(start + steps - 1) - g.first + 1;
            if (g.parts > 1 && g.first == me) {
                shared_item = make_int4(g.tok, g.n, g.kh, g.parts);
            }
            if (g.j1 > g.j0 && !publish(g)) break;
            item += steps + p.item_cost;
            at = item;
            i += tpc;
            if (i >= n) {
                i = 0;
                if (++kh == p.KVH) {
                    kh = 0;
                    do {
                        if (++seq >= p.b.batch) break;
                        s = seq_span(p.b, p.c, seq);
                        n = min(s.n, p.max_q);
                    } while (n == 0);
                }
            }
            if (item < end) steps = kv_steps(s.len - s.n + min(i + tpc, n) - 1, s.len);
        }
        if (lane == 0 && rank == 0) p.shared_items[me] = shared_item;
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
        // page and row of this lane's box of step j; a pair's CTA takes the boxes of its 64 slots for K
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
        auto load = [&](const CUtensorMap* map, bool is_k, uint32_t pos, int kh, int page, int row, int n) -> bool {
            const int first = PAIR && is_k ? rank * boxes / 2 : 0;  // this CTA's boxes: first .. first + count
            const int count = max(PAIR && is_k ? min(n - first, boxes / 2) : n, 0);
            const int cps = is_k ? P::kCps : P::kVCps;
            const int x0 = PAIR && !is_k ? rank * P::kVCps * 64 : 0;
            const uint32_t chunk = is_k ? P::kKChunk : kChunkBytes;
            for (int part = 0; part < P::kParts; ++part) {
                const uint32_t st = (pos + part) % P::kStages;
                ok = ok && !*bail.flag && bail.wait(&bars.empty[st], (((pos + part) / P::kStages) & 1) ^ 1);
                if (!__all_sync(kFull, ok)) return ok = false;
                if (lane == 0) {
                    if (count > 0)
                        mbar_expect_tx(&bars.full[st], static_cast<uint32_t>(count) * box_bytes * cps);
                    else
                        mbar_arrive(&bars.full[st]);
                }
                __syncwarp();
                if (lane >= first && lane < first + count) {
                    const uint32_t dst = smem_u32(ring + st * P::kStageBytes) + (lane - first) * box_bytes;
                    for (int ch = 0; ch < cps; ++ch)
                        tma_load_4d(dst + ch * chunk, map, x0 + (part * P::kCps + ch) * 64, p.order.pick(0, row, kh, page),
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
                const uint32_t bytes = static_cast<uint32_t>(p.box_tokens) * p.G * 128;
                mbar_expect_tx(&bars.q_full, bytes * NCH * NQ);
                for (int t = 0; t < NQ; ++t)
                    for (int ch = 0; ch < NCH; ++ch)
                        tma_load_3d_at(smem_u32(smem + (t * NCH + ch) * kChunkBytes), &tm_q, ch * 64, g.kh * p.G,
                                       g.tok + (t + rank) * p.tpt, &bars.q_full);
            }
            ++qs;
            for (int j = g.j0; j < g.j1 && ok; ++j, ++u) {
                int page, row, n;
                locate(g, j, page, row, n);
                if (NQ == 2) {
                    if (load(&tm_k, true, 2 * u * P::kParts, g.kh, page, row, n)) load(&tm_v, false, (2 * u + 1) * P::kParts, g.kh, page, row, n);
                } else {
                    if (load(&tm_k, true, (u == 0 ? 0 : 2 * u - 1) * P::kParts, g.kh, page, row, n) && u > 0)
                        load(&tm_v, false, 2 * u * P::kParts, vkh, vpage, vrow, vn);
                    vpage = page;
                    vrow = row;
                    vn = n;
                    vkh = g.kh;
                }
            }
        }
        if (NQ == 1 && ok && u > 0) load(&tm_v, false, 2 * u * P::kParts, vkh, vpage, vrow, vn);
        // No copy may still be landing when the CTA exits, and no commit's arrival may still be on its way (in a
        // pair, from the other CTA): nothing else waits for the last release of a stage, of Q or of a unit's P V.
        // A lane takes a stage, a unit's parity of a row tile, or Q: one after another the waits would add a
        // microsecond to the CTA's end.
        uint64_t *landed = nullptr, *released = nullptr;
        uint32_t phase = 0;
        if (lane < P::kStages) {
            if (pos_max > static_cast<uint32_t>(lane)) {
                // the last fill of this stage (a place that was skipped was filled one round earlier)
                uint32_t last = pos_max - 1 - (pos_max - 1 - lane) % P::kStages;
                if (NQ == 1 && u > 0 && last >= (2 * u - 1) * P::kParts && last < 2 * u * P::kParts) last -= P::kStages;
                if (static_cast<int>(last) >= 0) {
                    landed = &bars.full[lane];
                    released = &bars.empty[lane];
                    phase = last / P::kStages;
                }
            }
        } else if (lane < P::kStages + 2 * NQ) {
            const int i = lane - P::kStages;  // [row tile][parity]
            const uint32_t units = NQ == 2 ? u : (u + 1 - (i & 1)) / 2;
            if (units > 0) released = &bars.o_done[i >> 1][i & 1];
            phase = units - 1;
        } else if (lane == P::kStages + 2 * NQ && qs > 0) {
            landed = &bars.q_full;
            released = &bars.q_empty;
            phase = qs - 1;
        }
        if (landed) mbar_wait(landed, phase & 1);
        // (after a wait that gave up there is no knowing which arrivals will come)
        if (released && ok && !*bail.flag) bail.wait(released, phase & 1);
        __syncwarp();
    } else if (warp == kMmaWarp || warp == kMmaWarp + 1) {
        // ---- MMA: S(u) = Q K(u)^T once P of this buffer's previous unit has been used by O += P V ----
        const int w = warp - kMmaWarp;  // row tile (NQ = 2), or the parity of its units (NQ = 1)
        constexpr uint32_t id_qk = PAIR ? idesc_f16_pair<T>(kTile, false) : idesc_f16<T>(NQ == 2 ? kHalf : kTile, false);
        constexpr uint32_t id_pv = PAIR ? idesc_f16_pair<T>(NCH * 64, true) : idesc_f16<T>(P::kCps * 64, true);
        const uint32_t s_tm = tmem + w * kTile;
        const uint32_t o_tm = tmem + kO + (NQ == 2 ? w * NCH * 64 : 0);
        const uint32_t q_sm = smem_u32(smem) + (NQ == 2 ? w * NCH * kChunkBytes : 0);
        bool ok = true;
        // Both warps follow every fill of the ring in order, so a wait for a stage's phase
        // always comes after that stage's phase before (a parity wait that is a phase early
        // would return at once); a tile that is the other warp's is released unused.
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            // the flag only where the barrier is not complete: 2048 tokens over 16384 slots 478 -> 446 us, 4001-token
            // prompts of pairs 90.5 -> 87.5; a single row tile a CTA, which waits for HBM, has nothing from it (46.6, 47.7)
            if (NQ == 2 || PAIR)
                ok = ok && bail.ready(bar, parity);
            else
                ok = ok && !*bail.flag && bail.wait(bar, parity);
            return ok = __all_sync(kFull, ok);
        };
        auto tile_wait = [&](uint32_t pos) {
            for (int part = 0; part < P::kParts; ++part)
                if (!wait(&bars.full[(pos + part) % P::kStages], ((pos + part) / P::kStages) & 1) ||
                    (PAIR && rank == 0 && !wait(&bars.peer_full[(pos + part) % P::kStages], ((pos + part) / P::kStages) & 1)))
                    return false;
            return true;
        };
        auto tile_skip = [&](uint32_t pos) {
            if (!tile_wait(pos)) return;
            if (lane == 0)
                for (int part = 0; part < P::kParts; ++part) {
                    mbar_arrive(&bars.empty[(pos + part) % P::kStages]);
                    if (PAIR) mbar_arrive_at(&bars.empty[(pos + part) % P::kStages], 1);
                }
            __syncwarp();
        };
        auto v_pos = [&](uint32_t u) { return (NQ == 2 ? 2 * u + 1 : 2 * u + 2) * P::kParts; };
        auto k_pos = [&](uint32_t u) { return (NQ == 2 ? 2 * u : (u == 0 ? 0 : 2 * u - 1)) * P::kParts; };
        // clears the rows of slots past the sequence in V tile u (NQ = 2: both warps, the same zeros)
        auto clear = [&](uint32_t u, int valid) {
            if (valid >= kTile) return;
            for (int part = 0; part < P::kParts; ++part) {
                unsigned char* v = ring + ((v_pos(u) + part) % P::kStages) * P::kStageBytes;
                for (int e = valid * 8 + lane; e < kTile * 8; e += 32)
#pragma unroll
                    for (int ch = 0; ch < P::kVCps; ++ch)
                        *reinterpret_cast<uint4*>(v + ch * kChunkBytes + e * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async();
            __syncwarp();
        };
        // One thread's MMAs, back to back: a barrier test or a commit between them would hold the
        // tensor core up by 200 or 60 clocks.  Unit x is a kv step (NQ = 1), or half of one: the
        // weights and the V rows from 64 * half on.
        auto pv_mma = [&](uint32_t u, int half, bool first) {
            constexpr int kSteps = (NQ == 2 ? kHalf : kTile) / 16;
            const uint32_t p_tm = s_tm + half * kHalf;
#pragma unroll
            for (int part = 0; part < P::kParts; ++part) {
                const uint32_t v = smem_u32(ring + ((v_pos(u) + part) % P::kStages) * P::kStageBytes) + half * kHalf * 128;
#pragma unroll
                for (int kk = 0; kk < kSteps; ++kk)
                    if (PAIR)
                        mma_f16_ts_pair(o_tm, p_tm + kk * 8, desc_mn_major(v + kk * 2048, kChunkBytes), id_pv, !first || kk > 0);
                    else
                        mma_f16_ts(o_tm + part * P::kCps * 64, p_tm + kk * 8, desc_mn_major(v + kk * 2048, kChunkBytes), id_pv,
                               !first || kk > 0);
            }
        };
        auto qk_mma = [&](uint32_t u, int half) {
#pragma unroll
            for (int part = 0; part < P::kParts; ++part) {
                const uint32_t k = smem_u32(ring + ((k_pos(u) + part) % P::kStages) * P::kStageBytes) + half * kHalf * 128;
#pragma unroll
                for (int ch = 0; ch < P::kCps; ++ch)
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                        if (PAIR)
                            mma_f16_ss_pair(s_tm, desc_k_major(q_sm + ch * kChunkBytes + kk * 32),
                                            desc_k_major(k + ch * P::kKChunk + kk * 32), id_qk, ch + kk > 0);
                        else
                            mma_f16_ss(s_tm + half * kHalf, desc_k_major(q_sm + (part * P::kCps + ch) * kChunkBytes + kk * 32),
                                   desc_k_major(k + ch * kChunkBytes + kk * 32), id_qk, part + ch + kk > 0);
            }
        };
        auto commit = [&](uint64_t* bar) {
            if (PAIR)
                tc2_commit_both(bar);
            else
                tc1_commit(bar);
        };
        auto release = [&](uint32_t pos) {
            for (int part = 0; part < P::kParts; ++part) commit(&bars.empty[(pos + part) % P::kStages]);
        };
        uint32_t u = 0, segs = 0;
        Segment g;
        if (NQ == 2) {
            // S of half step x once the weights of half step x - 2, which lie in its place, have been used
            bool first[2] = {false, false};  // [half] of the step before: its first P V overwrites O
            int valid = kTile;
            auto pv = [&](uint32_t x) {
                const uint32_t v = x >> 1;
                const int half = static_cast<int>(x & 1);
                if (half == 0) {
                    if (!tile_wait(v_pos(v))) return false;
                    clear(v, valid);
                }
                if (!wait(&bars.p_full[w][half], v & 1)) return false;
                tc1_fence_after();
                if (lane == 0) pv_mma(v, half, first[half]);
                return true;
            };
            auto pv_done = [&](uint32_t x) {
                tc1_commit(&bars.o_done[w][x & 1]);
                if (x & 1) release(v_pos(x >> 1));
            };
            while (ok && next_seg(g)) {
                for (int j = g.j0; j < g.j1 && ok; ++j, ++u) {
                    for (int half = 0; half < 2 && ok; ++half) {
                        const uint32_t x = 2 * u + half;
                        if (u > 0 && !pv(x - 2)) break;
                        if (half == 0 && ((j == g.j0 && !wait(&bars.q_full, segs & 1)) || !tile_wait(k_pos(u)))) break;
                        tc1_fence_after();
                        if (lane == 0) {
                            qk_mma(u, half);
                            tc1_commit(&bars.s_full[w][half]);
                            if (u > 0) pv_done(x - 2);
                            if (half) release(k_pos(u));
                        }
                        __syncwarp();
                    }
                    first[0] = j == g.j0;
                    valid = max(min(g.len - j * kTile, kTile), 0);
                }
                if (!ok) break;
                if (lane == 0) tc1_commit(&bars.q_empty);  // through with the segment's Q
                __syncwarp();
                ++segs;
            }
            for (uint32_t x = 2 * u - 2; ok && u > 0 && x < 2 * u; ++x) {
                if (pv(x) && lane == 0) pv_done(x);
                __syncwarp();
            }
        } else if (PAIR && rank == 1) {
            // CTA 1 of a pair issues nothing: its first MMA warp passes each of its fills on to CTA 0, in the
            // ring's order, the V rows past the sequence cleared
            auto pass = [&](uint32_t pos) {
                if (lane == 0) mbar_arrive_at(&bars.peer_full[pos % P::kStages], 0);
                __syncwarp();
            };
            int valid = kTile;
            auto v = [&](uint32_t x) {
                if (!tile_wait(v_pos(x))) return;
                clear(x, valid);
                pass(v_pos(x));
            };
            while (ok && next_seg(g)) {
                if (w == 1) continue;
                if (!wait(&bars.q_full, segs & 1)) break;
                if (lane == 0) mbar_arrive_at(&bars.peer_q, 0);
                __syncwarp();
                for (int j = g.j0; j < g.j1 && ok; ++j, ++u) {
                    if (tile_wait(k_pos(u))) pass(k_pos(u));
                    if (u > 0 && ok) v(u - 1);
                    valid = max(min(g.len - j * kTile, kTile), 0);
                }
                ++segs;
            }
            if (ok && w == 0 && u > 0) v(u - 1);
        } else {
            auto q_wait = [&](uint32_t s) {
                return wait(&bars.q_full, s & 1) && (!PAIR || wait(&bars.peer_q, s & 1));
            };
            // S(u) once P(u - 2) has been used; the units of one parity are this warp's
            auto own = [&](uint32_t x) { return (x & 1) == static_cast<uint32_t>(w); };
            auto pv = [&](uint32_t x, bool first, int valid) {
                if (!own(x)) return tile_skip(v_pos(x));
                if (!tile_wait(v_pos(x))) return;
                clear(x, valid);
                if (!wait(&bars.p_full[0][w], (x >> 1) & 1)) return;
                // one O: the units take turns, each after the one before
                if (x > 0 && !wait(&bars.o_done[0][w ^ 1], ((x - 1) >> 1) & 1)) return;
                tc1_fence_after();
                if (lane == 0) {
                    pv_mma(x, 0, first);
                    commit(&bars.o_done[0][w]);
                    release(v_pos(x));
                }
                __syncwarp();
            };
            bool have = false, first = false;  // the unit before u: its P V is due
            int valid = kTile;
            while (ok && next_seg(g)) {
                bool fresh = true;  // the segment's Q has not been waited for
                for (int j = g.j0; j < g.j1 && ok; ++j, ++u) {
                    // in the ring's order: K(u) V(u - 1)
                    if (!own(u)) {
                        tile_skip(k_pos(u));
                    } else if ((!fresh || q_wait(segs)) && tile_wait(k_pos(u))) {
                        fresh = false;
                        tc1_fence_after();
                        if (lane == 0) {
                            qk_mma(u, 0);
                            commit(&bars.s_full[0][w]);
                            release(k_pos(u));
                        }
                        __syncwarp();
                    }
                    if (have && ok) pv(u - 1, first, valid);
                    have = true;
                    first = j == g.j0;
                    valid = max(min(g.len - j * kTile, kTile), 0);
                }
                // through with the segment's Q: a warp that had no unit in it comes after its load all the
                // same, or its arrival could count for the segment before
                if (ok && fresh) q_wait(segs);
                if (!ok) break;
                if (lane == 0) commit(&bars.q_empty);
                __syncwarp();
                ++segs;
            }
            if (ok && have) pv(u - 1, first, valid);
        }
    } else {
        // ---- softmax, one thread a row, and the output ----
        // NQ = 2: a warpgroup a row tile, 64 slots a unit.  NQ = 1: two warpgroups, 64 of a unit's 128 slots each.
        constexpr int kOut = 16;                              // columns of O in registers at a time
        constexpr int kUnits = NQ == 2 ? 2 : 1;               // units of a kv step
        const int grp = NQ == 2 ? warp >> 2 : 0, half = NQ == 2 ? 0 : warp >> 2, quarter = warp & 3;
        const int tile = PAIR ? rank : grp;  // row tile of the item
        const int r = quarter * 32 + lane;  // row of the tile
        const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t o_tm = tmem + lane_off + kO + grp * NCH * 64;
        const float c = p.scale * 1.44269504088896340736f;
        const int tok_in = r / p.G, head_in = r - tok_in * p.G;
        // this warp's columns of the output
        const int mid = (p.D / 2 + 15) / 16 * 16;
        const int d0 = half ? mid : 0, d1 = NQ == 2 || half ? p.D : mid;
        uint32_t u = 0;  // units so far of this group
        bool ok = true;
        // The other warp of these rows: a meeting, and x for its x.
        uint32_t turns = 0;
        auto meet = [&]() {
            tc1_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.pair[quarter]);
            ok = !*bail.flag && bail.wait(&bars.pair[quarter], turns & 1);
            ++turns;
            ok = __all_sync(kFull, ok);
            tc1_fence_after();
            return ok;
        };
        auto swap = [&](float x, float& other) {
            const int at = turns & 1;
            bars.xch[at][half][r] = x;
            if (!meet()) return false;
            other = bars.xch[at][half ^ 1][r];
            return true;
        };
        // O after unit x of this group
        auto o_wait = [&](uint32_t x) {
            ok = !*bail.flag && bail.wait(&bars.o_done[grp][x & 1], (x >> 1) & 1);
            ok = __all_sync(kFull, ok);
            if (ok) tc1_fence_after();
            return ok;
        };
        Segment g;
        while (ok && next_seg(g)) {
            const int toks = min(max(g.n - tile * p.tpt, 0), p.tpt);
            const bool live = tok_in < toks;  // (rows past tpt * G have tok_in >= tpt)
            const bool any_live = __any_sync(kFull, live);
            const int lim = live ? g.vis + tile * p.tpt + tok_in : -1;  // last slot this row sees
            int least = live ? lim : 0x7fffffff;
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) least = min(least, __shfl_xor_sync(kFull, least, off));
            const int h = g.kh * p.G + head_in;
            const int t = g.tok + tile * p.tpt + tok_in;
            if (p.gate && live && g.parts == 1) {
                // the gate is wanted at the segment's end: towards L2 now
                const char* at = reinterpret_cast<const char*>(p.gate + static_cast<size_t>(t) * p.gate_row +
                                                               static_cast<size_t>(h) * p.gate_head);
                for (int e = d0 * 4; e < d1 * 4; e += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(at + e));
            }
            float m = -INFINITY, l = 0.f;
            for (int j = g.j0 * kUnits; j < g.j1 * kUnits && ok; ++j, ++u) {
                ok = !*bail.flag && bail.wait(&bars.s_full[grp][u & 1], (u >> 1) & 1);
                if (!__all_sync(kFull, ok)) {
                    ok = false;
                    break;
                }
                tc1_fence_after();
                // The two row tiles' warps of one scheduler take turns at the exponentials: side by side
                // both would take twice as long and then leave the unit idle together.
                auto take_turn = [&]() {
                    if (NQ == 1 || (grp == 0 && u == 0)) return true;
                    ok = !*bail.flag && bail.wait(&bars.turn[grp][quarter], (grp == 0 ? u - 1 : u) & 1);
                    return ok = __all_sync(kFull, ok);
                };
                auto pass_turn = [&](uint32_t after) {
                    if (NQ == 2 && lane == 0) arrive_after(&bars.turn[grp ^ 1][quarter], after);
                };
                if (!any_live) {
                    if (!take_turn()) break;
                    pass_turn(0);
                } else {
                    // scores and weights of this thread: 64 columns, and 32 at the start of the unit's place
                    const uint32_t unit = tmem + lane_off + (NQ == 2 ? grp * kTile + (u & 1) * kHalf : (u & 1) * kTile);
                    const uint32_t s_tm = unit + half * kHalf, p_tm = unit + half * (kHalf / 2);
                    const int kv0 = NQ == 2 ? j * kHalf : j * kTile + half * kHalf;
                    float s[kHalf];
                    float mx = m;
#pragma unroll
                    for (int q = 0; q < kHalf; q += 32) tmem1_ld32(s_tm + q, s + q);
                    tmem1_wait_ld();
                    if (kv0 + kHalf - 1 > min(least, g.len - 1)) {
                        const int lm = min(lim, g.len - 1) - kv0;  // last column this row sees
#pragma unroll
                        for (int i = 0; i < kHalf; ++i)
                            if (i > lm) s[i] = -INFINITY;
                    }
                    float y0 = s[0], y1 = s[1], y2 = s[2];
#pragma unroll
                    for (int i = 0; i < kHalf; i += 8) {
                        mx = max3(mx, s[i], s[i + 1]);
                        y0 = max3(y0, s[i + 2], s[i + 3]);
                        y1 = max3(y1, s[i + 4], s[i + 5]);
                        y2 = max3(y2, s[i + 6], s[i + 7]);
                    }
                    mx = fmaxf(max3(mx, y0, y1), y2);
                    if (NQ == 1) {
                        // (the other warp has its scores, too, once this returns: its columns may be overwritten)
                        float other;
                        if (!swap(mx, other)) break;
                        mx = fmaxf(mx, other);
                    }
                    if (__any_sync(kFull, live && (mx - m) * c > kLazy)) {
                        const float f = mx == m ? 1.f : ex2((m - mx) * c);
                        m = mx;
                        l *= f;
                        if (j > g.j0 * kUnits) {
                            if (!o_wait(u - 1)) break;
#pragma unroll 1
                            for (int i = d0 / 16 * 16; i < (NQ == 2 || half ? NCH * 64 : mid); i += 16) {
                                float o[16];
                                tmem1_ld16(o_tm + i, o);
                                tmem1_wait_ld();
#pragma unroll
                                for (int e = 0; e < 16; ++e) o[e] *= f;
                                tmem1_st16(o_tm + i, reinterpret_cast<const uint32_t*>(o));
                            }
                        }
                    }
                    const float neg = m == -INFINITY ? 0.f : kLift<T> - m * c;
                    const float2 c2 = make_float2(c, c), neg2 = make_float2(neg, neg);
                    float2 l0 = make_float2(0.f, 0.f), l1 = make_float2(0.f, 0.f);
                    if (!take_turn()) break;
                    uint32_t w[kHalf / 2];
#pragma unroll
                    for (int i = 0; i < kHalf; i += 4) {
                        float2 a = __ffma2_rn(make_float2(s[i], s[i + 1]), c2, neg2);
                        float2 b = __ffma2_rn(make_float2(s[i + 2], s[i + 3]), c2, neg2);
                        a.x = ex2(a.x);
                        a.y = ex2(a.y);
                        b.x = ex2(b.x);
                        b.y = ex2(b.y);
                        l0 = __fadd2_rn(l0, a);
                        l1 = __fadd2_rn(l1, b);
                        w[i / 2] = Elem<T>::pack(a.x, a.y);
                        w[i / 2 + 1] = Elem<T>::pack(b.x, b.y);
                        if (i + 4 == kPass) pass_turn(w[i / 2 + 1]);
                    }
                    tmem1_st32(p_tm, w);
                    l += (l0.x + l0.y) + (l1.x + l1.y);
                    tmem1_wait_st();
                    tc1_fence_before();
                }
                __syncwarp();
                if (lane == 0) {
                    if (PAIR)
                        mbar_arrive_at(&bars.p_full[0][u & 1], 0);
                    else
                        mbar_arrive(&bars.p_full[grp][u & 1]);
                }
            }
            if (!ok) break;
            if (!o_wait(u - 1)) break;
            if (NQ == 1 && any_live) {
                float other;
                if (!swap(l, other) || !meet()) break;  // the second: both have read, the place may be written again
                l += other;
            }
            if (g.parts == 1) {
                if (any_live) {
                    const float inv = l == 0.f ? 0.f : 1.f / l;
                    // a chunk's gates are asked for a chunk ahead
                    float4 gate[2][kOut / 4];
                    auto ask = [&](int col, float4* to) {
                        if (!p.gate || !live || col >= d1) return;
#pragma unroll
                        for (int e = 0; e < kOut; e += 8)
                            if (col + e < d1) load_gate8(p, t, h, col + e, to + e / 4);
                    };
                    auto give = [&](int col, const float4* from) {
                        if (col >= d1) return;
                        float o[kOut];
#pragma unroll
                        for (int e = 0; e < kOut; e += 16) tmem1_ld16(o_tm + col + e, o + e);
                        tmem1_wait_ld();
                        if (live)
#pragma unroll
                            for (int e = 0; e < kOut; e += 8)
                                if (col + e < d1) put8<T>(p, t, h, col + e, o + e, inv, from + e / 4);
                        __syncwarp();
                    };
                    ask(d0, gate[0]);
#pragma unroll 1
                    for (int col = d0; col < d1; col += 2 * kOut) {
                        ask(col + kOut, gate[1]);
                        give(col, gate[0]);
                        ask(col + 2 * kOut, gate[0]);
                        give(col + kOut, gate[1]);
                    }
                    if (live && half == 0 && p.lse)
                        p.lse[static_cast<size_t>(t) * p.H + h] = lse_of<T>(m, p.scale, l);
                }
            } else if (any_live) {
                // a shared item: this CTA's part (neighbouring rows' 16 bytes lie side by side)
                const size_t sl = part_slot<P::kTiles>(me, g.first, tile);
                float4* dst = p.part + sl * (p.D / 4) * p.rows_cap + r;
                if (live && half == 0) p.ml[sl * p.rows_cap + r] = make_float2(m, l);
                dst += static_cast<size_t>(d0 / 4) * p.rows_cap;
#pragma unroll 1
                for (int col = d0; col < d1; col += 16) {
                    float o[16];
                    tmem1_ld16(o_tm + col, o);
                    tmem1_wait_ld();
                    if (live) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            dst[e * p.rows_cap] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                    }
                    dst += 4 * p.rows_cap;
                    __syncwarp();
                }
            }
            tc1_fence_before();
        }
    }

    tc1_fence_before();
    __syncthreads();
    if (PAIR) pair_sync();  // no CTA leaves while its peer's threads may still signal it (commits: the TMA warp's last waits)
    if (warp == kMmaWarp) {
        tc1_fence_after();
        if (PAIR)
            tmem2_dealloc(tmem, 512);
        else
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
                         int box_rows, const char* what) {
    struct Dim {
        int id;
        cuuint64_t count, stride;
        cuuint32_t box;
    } d[3] = {{0, static_cast<cuuint64_t>(c.page), static_cast<cuuint64_t>(c.row_stride) * 2,
               static_cast<cuuint32_t>(box_rows)},
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

// Pairs of CTAs that the current device runs at once (its SMs in twos, less where a cluster of SMs has an odd
// one), read once per device; half its SMs where that cannot be read.
int pair_count(int sms) {
    static std::atomic<int> counts[kMaxDevices];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return sms / 2;
    int n = counts[dev].load(std::memory_order_relaxed);
    if (n) return n;
    using Pl = Plan<4, 1, true>;
    static FuncAttr attr;
    if (ensure_smem(attn_tc_kernel<__half, 4, 1, true>, attr, Pl::kSmem, -1, "w4a8_attn_paged") != W4A8_OK) return sms / 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * (sms / 2));
    cfg.blockDim = dim3(Pl::kThreads);
    cfg.dynamicSmemBytes = Pl::kSmem;
    cudaLaunchAttribute a[1];
    a[0].id = cudaLaunchAttributeClusterDimension;
    a[0].val.clusterDim.x = 2;
    a[0].val.clusterDim.y = 1;
    a[0].val.clusterDim.z = 1;
    cfg.attrs = a;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, attn_tc_kernel<__half, 4, 1, true>, &cfg) != cudaSuccess || n < 1) {
        cudaGetLastError();
        n = sms / 2;
    }
    counts[dev].store(n, std::memory_order_relaxed);
    return n;
}

// How a call is laid out on the GPU, from its sizes alone.
struct Layout {
    int nch, nq, tpt, rows_cap, grid;  // grid: CTAs, or pairs of them
    bool pair;
    size_t items, slots, bytes;
};

Layout layout_of(int H, int KVH, int D, int batch, int max_q, int max_kv, int sms) {
    Layout x{};
    const int G = H / KVH;
    x.nch = (D + 63) / 64;
    x.tpt = kTile / G;
    // Two row tiles for each K and V tile where there are rows for both: in one CTA where O fits beside them, in
    // two for the widest heads, whose single CTAs would read 128 KB from L2 for 2048 clocks of MMA.
    const bool many = static_cast<long long>(max_q) * G > kTile;
    x.nq = many && x.nch <= 2 ? 2 : 1;
    x.pair = many && x.nch == 4;
    const int tiles_of = x.pair ? 2 : x.nq;
    x.rows_cap = std::min(x.tpt, std::max(max_q, 1)) * G;
    const long long tiles = (static_cast<long long>(std::max(max_q, 1)) + tiles_of * x.tpt - 1) / (tiles_of * x.tpt);
    const long long steps = std::max((static_cast<long long>(max_kv) + kTile - 1) / kTile, 1ll);
    const long long work = std::min(tiles * (steps + kGatedItemCost), 1ll << 20) * KVH * batch;  // the longest the line can be
    x.grid = static_cast<int>(std::min<long long>(x.pair ? pair_count(sms) : sms, work));
    x.items = (static_cast<size_t>(x.grid) * 16 + 255) / 256 * 256;
    x.slots = static_cast<size_t>(x.grid) * 2 * tiles_of * x.rows_cap;
    x.bytes = x.items + (x.slots * 8 + 255) / 256 * 256 + x.slots * D * 4;
    return x;
}

template <typename T, int NCH, int NQ, bool PAIR = false>
w4a8_status launch_tc(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const AttnParams& p, int grid,
                      cudaStream_t st) {
    using Pl = Plan<NCH, NQ, PAIR>;
    const char* what = "w4a8_attn_paged";
    static FuncAttr attr;
    const w4a8_status s = ensure_smem(attn_tc_kernel<T, NCH, NQ, PAIR>, attr, Pl::kSmem, -1, what);
    if (s != W4A8_OK) return s;
    const w4a8_status r = PAIR ? launch_cluster(what, attn_tc_kernel<T, NCH, NQ, PAIR>, dim3(2 * grid), dim3(Pl::kThreads),
                                                Pl::kSmem, 2, st, q, k, v, p)
                               : launch_pdl(what, attn_tc_kernel<T, NCH, NQ, PAIR>, dim3(grid), dim3(Pl::kThreads), Pl::kSmem,
                                            st, q, k, v, p);
    if (r != W4A8_OK || grid == 1) return r;
    // by how many threads a row's 8 columns are shared: few rows have many parts
    const int work = p.rows_cap * (p.D / 8);
    auto merge = [&](auto kernel, int pg) {
        const int per = kMergeThreads / pg;
        return launch_pdl(what, kernel, dim3(grid * Pl::kTiles, (work + per - 1) / per), dim3(kMergeThreads), 0, st, p);
    };
    if (p.rows_cap <= 16) return merge(attn_merge_kernel<T, Pl::kTiles, 16>, 16);
    if (p.rows_cap < 64) return merge(attn_merge_kernel<T, Pl::kTiles, 4>, 4);
    return merge(attn_merge_kernel<T, Pl::kTiles, 1>, 1);
}

template <typename T>
w4a8_status dispatch(int nch, int nq, bool pair, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                     const AttnParams& p, int grid, cudaStream_t st) {
    if (pair) return launch_tc<T, 4, 1, true>(q, k, v, p, grid, st);
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
    (void)tokens;  // partial results are a CTA's, not a token's
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
    p.item_cost = gate ? kGatedItemCost : kItemCost;
    p.box_rows = std::min(cache_box_rows(page), x.pair ? kTile / 2 : kTile);  // a pair's CTA takes 64 slots of K
    p.box_tokens = std::min(x.tpt, max_q);
    p.rows_cap = x.rows_cap;
    p.shared_items = static_cast<int4*>(workspace);
    p.ml = reinterpret_cast<float2*>(static_cast<char*>(workspace) + x.items);
    p.part = reinterpret_cast<float4*>(static_cast<char*>(workspace) + x.items + (x.slots * 8 + 255) / 256 * 256);
    p.err = device_error_word();
    CUtensorMap mq, mk, mv;
    st = encode_queries(&mq, q, dtype, H, D, q_row_stride, tokens, p.G, p.box_tokens, what);
    if (st == W4A8_OK) st = encode_cache(&mk, &p.order, k, p.c, KVH, D, p.box_rows, what);
    if (st == W4A8_OK) st = encode_cache(&mv, &p.order, v, p.c, KVH, D, p.box_rows, what);
    if (st != W4A8_OK) return st;
    cudaStream_t cs = static_cast<cudaStream_t>(stream);
    return dtype == W4A8_F16 ? dispatch<__half>(x.nch, x.nq, x.pair, mq, mk, mv, p, x.grid, cs)
                             : dispatch<__nv_bfloat16>(x.nch, x.nq, x.pair, mq, mk, mv, p, x.grid, cs);
}

}  // extern "C"
