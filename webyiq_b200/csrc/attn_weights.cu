// The attention weight that each cached slot received from the step's new tokens,
// added to what it had:
//
//   acc[b, kvh, j] += sum over new tokens i that see j, query heads h of kvh, of
//                     exp(scale q_ih . k_j - lse_ih)
//
// The scores come from the tensor cores the other way round, S^T = K Q^T: a tile's 128
// slots are the MMA's M (a tensor memory lane and a thread each), the query rows (token
// * G + head) its N.  So a slot's sum over rows stays in one thread, in a fixed order:
// no atomics and no shuffles, the same bits every time.  The exponent's offset is per
// column, read from shared memory (one broadcast load for four).
//
// An item is one tile of slots of a kv head; it stays in shared memory while the query
// rows that see it pass.  Items lie on a line, each as long as its row tiles and one for
// the tile itself, and each CTA takes an equal stretch of it, found on the device from
// the batch's lengths.  An item that a stretch boundary cuts leaves its parts' sums in the
// workspace, and a small kernel adds those in the order of the stretches.  Single tokens
// are bound by HBM (K is read once), chunks by the exponentials: 128 x 128 of them take
// the SM's 16 a clock 1024 clocks, the MMA half of that at 128-wide heads.  Measured: 1500
// tokens over 8200 slots, 32 / 8 heads of 128, in 134 us at best, 139 to 142 usually (682 TFLOP/s, the
// exponentials alone take 151 K clocks, 77 us at 1965 MHz; 182 with one MMA warp, whose barrier tests and commits left gaps, 251
// with two softmax warpgroups); 16 single tokens over 56 MB in 17.6 to 18.8 us.
// (136 and 17.9 with the abort flag read before every wait, not only where one has to wait.)
//
// Warp roles: four softmax warpgroups that take row tiles in turn, an S buffer each, so
// that one's waits and loads run beside the others' exponentials (two left the unit idle
// half of the time), then TMA, MMA, and the warp that walks the line.
#include <algorithm>

#include "launch.cuh"
#include "tc_f16.cuh"

namespace w4a8 {

namespace {

constexpr int kTile = 128;
constexpr uint32_t kChunkBytes = kTile * 128;  // 128 rows x 64 elements
constexpr int kRing = 13 * kChunkBytes;         // tiles of slots, then tiles of query rows
constexpr int kMaxStages = 8;
constexpr int kGroups = 4, kItems = 4;
constexpr int kSoftWarps = 4 * kGroups, kThreads = (kSoftWarps + 4) * 32;

struct WeightParams {
    int H, KVH, G, nch;
    int tpt;         // tokens of a row tile
    int box_tokens;  // tokens that one load of query rows brings
    int cols;        // N of the MMA: box_tokens * G rounded up to 16
    uint32_t k_stages, q_stages;
    uint32_t k_bytes, q_bytes;  // of a tile in the ring
    float scale;
    const float* lse;
    float* acc;
    int acc_stride, max_q;
    int box_rows;
    CacheOrder order;
    int4* shared_items;  // [CTA] the item that starts in its stretch and goes on in the next: row, tile, slots, parts
    float* part;         // [CTA][2][128]
    unsigned int* err;
    PagedCache c;
    PagedBatch b;
};

struct Item {
    int seq, kh;
    int t0, n;      // the sequence's first new token (global) and how many
    int vis;        // last slot its first new token sees
    int len, j;     // slots, and the tile's number
    int i0, steps;  // row tiles, of those that see something of the slots; steps == 0: the end
    int first, parts;  // first CTA of the item, CTAs that share it
};

struct Smem {
    unsigned char ring[kRing];
    float off[kGroups][2][kTile];      // [group][turn][column]: -lse * log2 e
    float sum[2][kGroups - 1][kTile];  // [turn]: the other groups' sums of an item, on the way to the first
    uint64_t k_full[kMaxStages], k_empty[kMaxStages], q_full[kMaxStages], q_empty[kMaxStages];
    uint64_t s_full[kGroups], s_empty[kGroups];
    uint64_t item_full[kItems], item_empty[kItems];
    uint64_t group[kGroups], sum_full[2], sum_empty[2];
    Item item[kItems];
    uint32_t tmem;
    int abort;
};
constexpr size_t kSmemBytes = 1024 + sizeof(Smem);
static_assert(kSmemBytes <= 227 * 1024, "shared memory plan exceeds 227 KB");

// First row tile of a sequence that sees slot tile j (the rows before it see none of it).
__device__ __forceinline__ int first_row_tile(const SeqSpan& s, int j, int tpt) {
    return max(0, j * kTile - (s.len - s.n)) / tpt;
}

// A CTA's part of the item that starts in its stretch lies second, of the one that came over first.
__device__ __forceinline__ size_t part_at(int cta, int first) {
    return (static_cast<size_t>(cta) * 2 + (cta == first ? 1 : 0)) * kTile;
}

__global__ void __launch_bounds__(kTile) weights_merge_kernel(const WeightParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int first = blockIdx.x;
    const int4 item = ld_dep(p.shared_items + first);
    const int slot = item.y * kTile + threadIdx.x;
    if (item.w == 0 || slot >= item.z) return;
    float total = 0.f;
    for (int q = 0; q < item.w; ++q) total += ld_dep(p.part + part_at(first + q, first) + threadIdx.x);
    float* at = p.acc + static_cast<size_t>(item.x) * p.acc_stride + slot;
    *at = ld_dep(at) + total;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
    weights_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                      const WeightParams p) {
    extern __shared__ unsigned char smem_raw[];
    Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kTmaWarp = kSoftWarps, kMmaWarp = kTmaWarp + 1, kLineWarp = kTmaWarp + 3;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kMaxStages; ++i) {
            mbar_init(&sm.k_full[i], 1);
            mbar_init(&sm.k_empty[i], 2);  // both MMA warps, whether they use the tile or not
            mbar_init(&sm.q_full[i], 1);
            mbar_init(&sm.q_empty[i], 2);
        }
        for (int i = 0; i < kGroups; ++i) {
            mbar_init(&sm.s_full[i], 1);
            mbar_init(&sm.s_empty[i], 4);
            mbar_init(&sm.group[i], 128);
        }
        for (int i = 0; i < kItems; ++i) {
            mbar_init(&sm.item_full[i], 1);
            mbar_init(&sm.item_empty[i], kSoftWarps + 3);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sm.sum_full[i], kSoftWarps - 4);
            mbar_init(&sm.sum_empty[i], 4);
        }
        sm.abort = 0;
        mbar_init_fence();
    }
    if (warp == kMmaWarp) tmem1_alloc(&sm.tmem, 512);
    tc1_fence_before();
    __syncthreads();
    tc1_fence_after();
    const uint32_t tmem = sm.tmem;
    pdl_launch_dependents();
    pdl_wait();

    const Bail bail{&sm.abort, p.err};
    uint32_t items = 0;
    auto next_item = [&](Item& it) -> bool {
        const uint32_t i = items % kItems;
        const bool ok = bail.ready(&sm.item_full[i], (items / kItems) & 1);
        if (!__all_sync(kFull, ok)) return false;
        it = sm.item[i];
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.item_empty[i]);
        ++items;
        return it.steps > 0;
    };

    if (warp == kLineWarp) {
        // ---- the line of items: an item's length is its row tiles and one for its slots ----
        // new tokens and slot tiles of sequence b; none where either is none
        auto span = [&](int b, SeqSpan& s, int& n, int& tiles) {
            s = b < p.b.batch ? seq_span(p.b, p.c, b) : SeqSpan{};
            n = min(s.n, p.max_q);
            const int slots = n > 0 ? min(s.len, p.acc_stride) : 0;
            tiles = slots / kTile + (slots % kTile != 0);
        };
        auto item_len = [&](const SeqSpan& s, int n, int j) {
            return max((n + p.tpt - 1) / p.tpt - first_row_tile(s, j, p.tpt), 0) + 1;
        };
        // length of this lane's sequence, all its kv heads
        auto seq_len = [&](const SeqSpan& s, int n, int tiles) {
            const bool many = n > p.tpt || n < s.n;
            long long total = tiles * 2ll;  // one row tile, which sees something of every slot tile
            for (unsigned todo = __ballot_sync(kFull, many); todo; todo &= todo - 1) {
                const int src = __ffs(todo) - 1;
                SeqSpan o;
                o.t0 = 0;
                o.n = __shfl_sync(kFull, s.n, src);
                o.len = __shfl_sync(kFull, s.len, src);
                const int on = __shfl_sync(kFull, n, src), ot = __shfl_sync(kFull, tiles, src);
                long long sum = 0;
                for (int j = lane; j < ot; j += 32) sum += item_len(o, on, j);
                sum = line_sum(sum);
                if (lane == src) total = sum;
            }
            return line_heads(total, p.KVH);
        };
        SeqSpan s;
        int n, tiles;
        int mine = 0;
        long long whole = 0;
        for (int b0 = 0; b0 < p.b.batch; b0 += 32) {
            span(b0 + lane, s, n, tiles);
            const long long places = seq_len(s, n, tiles);
            whole += line_sum(places);
            mine = static_cast<int>(places);  // (used where the whole fits)
        }
        const int total = line_length(whole, p.err);
        const int ctas = min(static_cast<int>(gridDim.x), total), me = blockIdx.x;
        int at = 0, end = 0;
        if (me < ctas) {
            at = line_mul_div(me, total, ctas);
            end = line_mul_div(me + 1, total, ctas);
        }
        // the CTA whose stretch holds place x
        auto cta_of = [&](int x) { return line_mul_div(x + 1, ctas, total, 1); };
        int seq = 0, kh = 0, j = 0;
        int pos = 0;  // start of item (seq, kh, j)
        bool ok = true;
        if (at < end) {
            for (int b0 = 0; b0 < p.b.batch; b0 += 32) {
                if (p.b.batch > 32) {  // (one round: as above)
                    span(b0 + lane, s, n, tiles);
                    mine = static_cast<int>(seq_len(s, n, tiles));
                }
                int upto = mine;
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) {
                    const int y = __shfl_up_sync(kFull, upto, off);
                    if (lane >= off) upto += y;
                }
                const unsigned past = __ballot_sync(kFull, pos + upto > at);
                if (past) {
                    const int f = __ffs(past) - 1;
                    seq = b0 + f;
                    pos += __shfl_sync(kFull, upto - mine, f);
                    const int per = __shfl_sync(kFull, mine, f) / p.KVH;
                    kh = (at - pos) / per;
                    pos += kh * per;
                    s = SeqSpan{__shfl_sync(kFull, s.t0, f), __shfl_sync(kFull, s.n, f), __shfl_sync(kFull, s.len, f)};
                    n = __shfl_sync(kFull, n, f);
                    tiles = __shfl_sync(kFull, tiles, f);
                    break;
                }
                pos += __shfl_sync(kFull, upto, 31);
            }
            // the item that holds place `at`
            for (int j0 = 0; j0 < tiles; j0 += 32) {
                const int len = j0 + lane < tiles ? item_len(s, n, j0 + lane) : 0;
                int upto = len;
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) {
                    const int y = __shfl_up_sync(kFull, upto, off);
                    if (lane >= off) upto += y;
                }
                const unsigned past = __ballot_sync(kFull, pos + upto > at);
                if (past) {
                    const int f = __ffs(past) - 1;
                    j = j0 + f;
                    pos += __shfl_sync(kFull, upto - len, f);
                    break;
                }
                j = min(j0 + 32, tiles);
                pos += __shfl_sync(kFull, upto, 31);
            }
        }
        uint32_t sent = 0;
        auto publish = [&](const Item& it) {
            const uint32_t i = sent % kItems;
            ok = ok && bail.ready(&sm.item_empty[i], ((sent / kItems) & 1) ^ 1);
            if (!__all_sync(kFull, ok)) return ok = false;
            if (lane == 0) {
                sm.item[i] = it;
                mbar_arrive(&sm.item_full[i]);
            }
            ++sent;
            return true;
        };
        int4 shared_item = make_int4(0, 0, 0, 0);
        while (ok && pos < end) {
            if (j >= tiles) {  // the next kv head or sequence
                j = 0;
                if (++kh == p.KVH) {
                    kh = 0;
                    do {
                        if (++seq >= p.b.batch) break;
                        span(seq, s, n, tiles);
                    } while (tiles == 0);
                    if (seq >= p.b.batch) break;
                }
            }
            Item it;
            it.seq = seq;
            it.kh = kh;
            it.t0 = s.t0;
            it.n = n;
            it.vis = s.len - s.n;
            it.len = min(s.len, p.acc_stride);
            it.j = j;
            const int i0 = first_row_tile(s, j, p.tpt), steps = max((n + p.tpt - 1) / p.tpt - i0, 0);
            const int start = pos + 1;
            const int lo = max(at - start, 0), hi = min(steps, end - start);
            it.i0 = i0 + lo;
            it.steps = hi - lo;
            if (hi > lo) {
                it.first = cta_of(start);
                it.parts = cta_of(start + steps - 1) - it.first + 1;
                if (it.parts > 1 && it.first == static_cast<int>(blockIdx.x))
                    shared_item = make_int4(seq * p.KVH + kh, j, it.len, it.parts);
                if (!publish(it)) break;
            }
            pos += steps + 1;
            at = pos;
            ++j;
        }
        if (lane == 0 && p.shared_items) p.shared_items[blockIdx.x] = shared_item;
        Item stop{};
        if (ok) publish(stop);
    } else if (warp == kTmaWarp) {
        // ---- TMA: the item's slots, then the query rows, chunk by chunk ----
        const int boxes = kTile / p.box_rows;
        const uint32_t box_bytes = static_cast<uint32_t>(p.box_rows) * 128;
        const uint32_t q_load = static_cast<uint32_t>(p.box_tokens) * p.G * 128;  // a chunk's bytes
        uint32_t kn = 0, qn = 0;
        bool ok = true;
        // page and row of this lane's box of an item: looked up an item ahead
        auto locate = [&](const Item& it, int& page, int& row, int& n) {
            const int s0 = it.j * kTile + lane * p.box_rows;
            n = min(boxes, (it.len - it.j * kTile + p.box_rows - 1) / p.box_rows);
            page = row = 0;
            if (lane < n) {
                const int pi = s0 / p.c.page;
                page = static_cast<int>(page_of(p.b, p.c, it.seq, pi));
                row = s0 - pi * p.c.page;
            }
        };
        Item it, next;
        int page = 0, row = 0, n = 0, page_next = 0, row_next = 0, n_next = 0;
        bool more = next_item(it);
        if (more) locate(it, page, row, n);
        for (; ok && more; it = next, page = page_next, row = row_next, n = n_next) {
            more = next_item(next);
            if (more) locate(next, page_next, row_next, n_next);
            const uint32_t ks = kn % p.k_stages;
            ok = bail.ready(&sm.k_empty[ks], ((kn / p.k_stages) & 1) ^ 1);
            if (!(ok = __all_sync(kFull, ok))) break;
            if (lane == 0) mbar_expect_tx(&sm.k_full[ks], static_cast<uint32_t>(n) * box_bytes * p.nch);
            __syncwarp();
            if (lane < n)
                for (int ch = 0; ch < p.nch; ++ch)
                    tma_load_4d(smem_u32(sm.ring) + ks * p.k_bytes + ch * kChunkBytes + lane * box_bytes, &tm_k, ch * 64,
                                p.order.pick(0, row, it.kh, page), p.order.pick(1, row, it.kh, page),
                                p.order.pick(2, row, it.kh, page), &sm.k_full[ks]);
            ++kn;
            for (int i = it.i0; i < it.i0 + it.steps; ++i, ++qn) {
                const uint32_t qs = qn % p.q_stages;
                ok = bail.ready(&sm.q_empty[qs], ((qn / p.q_stages) & 1) ^ 1);
                if (!(ok = __all_sync(kFull, ok))) break;
                if (lane == 0) mbar_expect_tx(&sm.q_full[qs], q_load * p.nch);
                __syncwarp();
                if (lane < p.nch)
                    tma_load_3d_at(smem_u32(sm.ring) + p.k_stages * p.k_bytes + qs * p.q_bytes + lane * (p.q_bytes / p.nch), &tm_q,
                                   lane * 64, it.kh * p.G, it.t0 + i * p.tpt, &sm.q_full[qs]);
            }
        }
        // no copy may still be landing when the CTA exits, and no commit's arrival (the last releases of the stages,
        // which nothing else waits for) still be on its way: a lane takes a stage
        const bool of_q = lane >= kMaxStages;
        const uint32_t stage = of_q ? lane - kMaxStages : lane, stages = of_q ? p.q_stages : p.k_stages, fills = of_q ? qn : kn;
        if (stage < stages && stage < fills) {
            const uint32_t last = (fills - 1 - stage) / stages;  // its last fill's phase
            mbar_wait(of_q ? &sm.q_full[stage] : &sm.k_full[stage], last & 1);
            // (after a wait that gave up there is no knowing which arrivals will come)
            if (ok && !*bail.flag) bail.wait(of_q ? &sm.q_empty[stage] : &sm.k_empty[stage], last & 1);
        }
        __syncwarp();
    } else if (warp == kMmaWarp || warp == kMmaWarp + 1) {
        // ---- MMA: S^T = K Q^T, the even row tiles from one warp and the odd ones from the other (a barrier
        //      test or a commit holds up its own thread's MMAs only).  Both follow every fill in order. ----
        const uint32_t w = static_cast<uint32_t>(warp - kMmaWarp);
        const uint32_t idesc = idesc_f16<T>(0, false) | (static_cast<uint32_t>(p.cols >> 3) << 17);
        uint32_t kn = 0, sn = 0;
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            ok = ok && bail.ready(bar, parity);
            return ok = __all_sync(kFull, ok);
        };
        Item it;
        while (ok && next_item(it)) {
            const uint32_t ks = kn % p.k_stages;
            if (!wait(&sm.k_full[ks], (kn / p.k_stages) & 1)) break;
            const uint32_t ka = smem_u32(sm.ring) + ks * p.k_bytes;
            for (int i = 0; i < it.steps; ++i, ++sn) {
                const uint32_t qs = sn % p.q_stages, buf = sn % kGroups;
                if (!wait(&sm.q_full[qs], (sn / p.q_stages) & 1)) break;
                if ((sn & 1) != w) {
                    if (lane == 0) mbar_arrive(&sm.q_empty[qs]);
                    __syncwarp();
                    continue;
                }
                if (!wait(&sm.s_empty[buf], ((sn / kGroups) & 1) ^ 1)) break;
                tc1_fence_after();
                if (lane == 0) {
                    const uint32_t qa = smem_u32(sm.ring) + p.k_stages * p.k_bytes + qs * p.q_bytes, qc = p.q_bytes / p.nch;
                    for (int ch = 0; ch < p.nch; ++ch)
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            mma_f16_ss(tmem + buf * kTile, desc_k_major(ka + ch * kChunkBytes + kk * 32),
                                       desc_k_major(qa + ch * qc + kk * 32), idesc, ch + kk > 0);
                    tc1_commit(&sm.s_full[buf]);
                    tc1_commit(&sm.q_empty[qs]);
                }
                __syncwarp();
            }
            if (lane == 0 && ok) tc1_commit(&sm.k_empty[ks]);
            __syncwarp();
            ++kn;
        }
    } else if (warp < kSoftWarps) {
        // ---- exponentials and sums, one thread a slot ----
        const int grp = warp >> 2, gt = threadIdx.x & 127;
        const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const float c = p.scale * 1.44269504088896340736f;
        const float2 c2 = make_float2(c, c);
        const int tok_in = gt / p.G, head_in = gt - tok_in * p.G;  // this thread's column when offsets are fetched
        uint32_t sn = 0, turn = 0, done = 0;
        bool ok = true;
        // this thread's column's offset in row tile i of an item: asked for a tile ahead
        auto offset = [&](const Item& it, int i) {
            const int tok = (it.i0 + i) * p.tpt + tok_in;
            if (i >= it.steps || tok_in >= p.tpt || tok >= it.n) return 0.f;
            return ld_dep(p.lse + static_cast<size_t>(it.t0 + tok) * p.H + it.kh * p.G + head_in);
        };
        // the first row tile of an item that is this group's, if the item's first is number s of all
        auto first = [&](uint32_t s) { return static_cast<int>((static_cast<uint32_t>(grp) - s) % kGroups); };
        Item it, next;
        bool more = next_item(it);
        float pre = more ? offset(it, first(sn)) : 0.f;
        while (more && ok) {
            more = next_item(next);
            const int i_first = first(sn), i_next = first(sn + it.steps);
            const float pre_next = more ? offset(next, i_next) : 0.f;
            const int slot = it.j * kTile + gt;
            float total = 0.f;
            for (int i = i_first; i < it.steps && ok; i += kGroups) {
                const int tok0 = (it.i0 + i) * p.tpt;
                const int toks = min(it.n - tok0, p.tpt);
                // offsets of the tile's columns, for the whole group
                float* off = sm.off[grp][turn & 1];
                off[gt] = pre * -1.44269504088896340736f;
                pre = offset(it, i + kGroups);
                mbar_arrive(&sm.group[grp]);
                ok = bail.ready(&sm.group[grp], turn & 1);
                ++turn;
                ok = ok && bail.ready(&sm.s_full[grp], ((sn + i) / kGroups) & 1);
                if (!(ok = __all_sync(kFull, ok))) break;
                tc1_fence_after();
                const uint32_t s_tm = tmem + lane_off + grp * kTile;
                const int cols = toks * p.G;
                // the first column that sees this slot
                const int lo = max(slot - (it.vis + tok0), 0) * p.G;
                float2 a0 = make_float2(0.f, 0.f), a1 = make_float2(0.f, 0.f);
                auto add = [&](const float* s, int x, int e, bool masked) {
                    const float4 o = *reinterpret_cast<const float4*>(off + x + e);
                    float2 u = __ffma2_rn(make_float2(s[e], s[e + 1]), c2, make_float2(o.x, o.y));
                    float2 v = __ffma2_rn(make_float2(s[e + 2], s[e + 3]), c2, make_float2(o.z, o.w));
                    u.x = ex2(u.x);
                    u.y = ex2(u.y);
                    v.x = ex2(v.x);
                    v.y = ex2(v.y);
                    if (masked) {
                        const int q = x + e;
                        u.x = q >= lo && q < cols ? u.x : 0.f;
                        u.y = q + 1 >= lo && q + 1 < cols ? u.y : 0.f;
                        v.x = q + 2 >= lo && q + 2 < cols ? v.x : 0.f;
                        v.y = q + 3 >= lo && q + 3 < cols ? v.y : 0.f;
                    }
                    a0 = __fadd2_rn(a0, u);
                    a1 = __fadd2_rn(a1, v);
                };
                if (cols == kTile && __all_sync(kFull, lo == 0)) {
                    // every column is live and sees every slot of the warp
#pragma unroll 1
                    for (int x = 0; x < kTile; x += 32) {
                        float s[32];
                        tmem1_ld32(s_tm + x, s);
                        tmem1_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; e += 4) add(s, x, e, false);
                    }
                } else {
#pragma unroll 1
                    for (int x = 0; x < cols; x += 16) {
                        float s[16];
                        tmem1_ld16(s_tm + x, s);
                        tmem1_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; e += 4) add(s, x, e, true);
                    }
                }
                total += (a0.x + a0.y) + (a1.x + a1.y);
                tc1_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.s_empty[grp]);
            }
            if (!ok) break;
            bool writes = i_first == 0;  // a single row tile: the group that has it
            if (it.steps > 1) {
                // the other groups hand their shares of the item to the first
                const uint32_t d = done & 1, phase = (done >> 1) & 1;
                ++done;
                ok = bail.ready(grp ? &sm.sum_empty[d] : &sm.sum_full[d], grp ? phase ^ 1 : phase);
                if (!(ok = __all_sync(kFull, ok))) break;
                if (grp)
                    sm.sum[d][grp - 1][gt] = total;
                else
#pragma unroll
                    for (int x = 0; x < kGroups - 1; ++x) total += sm.sum[d][x][gt];
                __syncwarp();
                if (lane == 0) mbar_arrive(grp ? &sm.sum_full[d] : &sm.sum_empty[d]);
                writes = grp == 0;
            }
            if (writes) {
                if (it.parts > 1) {
                    p.part[part_at(blockIdx.x, it.first) + gt] = total;
                } else if (slot < it.len) {
                    float* at = p.acc + (static_cast<size_t>(it.seq) * p.KVH + it.kh) * p.acc_stride + slot;
                    *at = ld_dep(at) + total;
                }
            }
            sn += it.steps;
            it = next;
            pre = pre_next;
        }
    }

    tc1_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc1_fence_after();
        tmem1_dealloc(tmem, 512);
    }
}

}  // namespace

int sm_count();  // capi.cu

}  // namespace w4a8

using namespace w4a8;

extern "C" {

W4A8_API size_t w4a8_attn_weights_workspace_bytes(int32_t H, int32_t KVH, int32_t max_q) {
    // a row tile takes all the query rows of a kv head: no item is cut
    if (H < 1 || KVH < 1 || static_cast<long long>(H / KVH) * max_q <= kTile) return 0;
    return static_cast<size_t>(sm_count()) * (sizeof(int4) + 2 * kTile * sizeof(float));
}

W4A8_API w4a8_status w4a8_attn_weights(const void* q, int32_t q_row_stride, const float* lse, int32_t H, int32_t KVH,
                                       int32_t D, float scale, const uint32_t* q_start, const uint32_t* kv_len,
                                       const uint32_t* table, int32_t batch, int32_t table_stride, int32_t tokens,
                                       int32_t max_q, int32_t max_kv, const void* k, int32_t dtype, int32_t pages,
                                       int32_t page, size_t page_stride, int32_t head_stride, int32_t row_stride,
                                       float* acc, int32_t acc_stride, void* workspace, size_t workspace_bytes,
                                       void* stream) {
    const char* what = "w4a8_attn_weights";
    WeightParams p{};
    p.c = PagedCache{const_cast<void*>(k), const_cast<void*>(k), dtype, pages, page, page_stride, head_stride, row_stride};
    p.b = PagedBatch{q_start, kv_len, table, batch, table_stride, tokens};
    w4a8_status st = check_heads(what, H, KVH, D);
    if (st == W4A8_OK) st = check_cache(what, p.c, KVH, D);
    if (st == W4A8_OK) st = check_batch(what, p.b);
    if (st != W4A8_OK) return st;
    if (static_cast<long long>(table_stride) * page >= (1ll << 31))
        return set_error(W4A8_EINVAL, "%s: %d pages of %d slots a sequence", what, table_stride, page);
    if (tokens > 0 && (!q || !lse || !acc)) return set_error(W4A8_EINVAL, "%s: NULL pointer", what);
    if (!aligned(q, 16) || !aligned(acc, 4) || !aligned(lse, 4))
        return set_error(W4A8_EINVAL, "%s: q must be 16-byte aligned, lse and acc 4-byte", what);
    if (q_row_stride % 8 || q_row_stride < static_cast<long long>(H) * D)
        return set_error(W4A8_EINVAL, "%s: q row stride %d (a multiple of 8 that holds the heads)", what, q_row_stride);
    if (max_q < 0 || max_q > (1 << 24) || max_kv < 0 || acc_stride < max_kv)
        return set_error(W4A8_EINVAL, "%s: max_q=%d max_kv=%d, %d weights a head", what, max_q, max_kv, acc_stride);
    if (!(scale > 0.f) || scale > 1e30f) return set_error(W4A8_EINVAL, "%s: scale %g", what, scale);
    if (tokens == 0 || max_q == 0 || max_kv == 0) return W4A8_OK;
    p.H = H;
    p.KVH = KVH;
    p.G = H / KVH;
    p.nch = (D + 63) / 64;
    p.tpt = kTile / p.G;
    p.box_tokens = max_q < p.tpt ? max_q : p.tpt;
    p.cols = (p.box_tokens * p.G + 15) / 16 * 16;
    // the ring: two to four tiles of query rows (all they can use where they are few), slots in the rest
    p.k_bytes = p.nch * kChunkBytes;
    p.q_bytes = p.nch * p.cols * 128;
    p.q_stages = std::min<uint32_t>(4, std::max<uint32_t>(2, kRing / 2 / p.q_bytes));
    p.k_stages = std::min<uint32_t>(kMaxStages, (kRing - p.q_stages * p.q_bytes) / p.k_bytes);
    p.scale = scale;
    p.lse = lse;
    p.acc = acc;
    p.acc_stride = acc_stride;
    p.max_q = max_q;
    p.box_rows = cache_box_rows(page);
    p.err = device_error_word();
    const size_t need = w4a8_attn_weights_workspace_bytes(H, KVH, max_q);
    if (need && (!workspace || !aligned(workspace, 16) || workspace_bytes < need))
        return set_error(W4A8_EINVAL, "%s: workspace NULL, misaligned or under %zu bytes", what, need);
    p.shared_items = need ? static_cast<int4*>(workspace) : nullptr;
    p.part = need ? reinterpret_cast<float*>(p.shared_items + sm_count()) : nullptr;
    CUtensorMap mq, mk;
    st = encode_queries(&mq, q, dtype, H, D, q_row_stride, tokens, p.G, p.box_tokens, what);
    if (st == W4A8_OK) st = encode_cache(&mk, &p.order, k, p.c, KVH, D, p.box_rows, what);
    if (st != W4A8_OK) return st;
    // as many CTAs as the line can have places
    const long long tiles = (static_cast<long long>(max_kv) + kTile - 1) / kTile;
    const long long rows = (static_cast<long long>(max_q) + p.tpt - 1) / p.tpt;
    const long long most = std::min(tiles * (need ? rows + 1 : 1), 1ll << 20) * KVH * batch;
    const int grid = static_cast<int>(std::min<long long>(most, sm_count()));
    cudaStream_t cs = static_cast<cudaStream_t>(stream);
    static FuncAttr a16, ab16;
    if (dtype == W4A8_F16) {
        st = ensure_smem(weights_tc_kernel<__half>, a16, kSmemBytes, -1, what);
        if (st == W4A8_OK) st = launch_pdl(what, weights_tc_kernel<__half>, dim3(grid), dim3(kThreads), kSmemBytes, cs, mq, mk, p);
    } else {
        st = ensure_smem(weights_tc_kernel<__nv_bfloat16>, ab16, kSmemBytes, -1, what);
        if (st == W4A8_OK)
            st = launch_pdl(what, weights_tc_kernel<__nv_bfloat16>, dim3(grid), dim3(kThreads), kSmemBytes, cs, mq, mk, p);
    }
    if (st != W4A8_OK || !need || grid == 1) return st;
    return launch_pdl(what, weights_merge_kernel, dim3(grid), dim3(kTile), 0, cs, p);
}

}  // extern "C"
