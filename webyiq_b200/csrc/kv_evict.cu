// Eviction from the paged cache by accumulated attention weight.
//
// Per sequence and kv head, of `len` slots the n = min(len, keep) first of this order
// stay: the protected ones (position below `sink`, or from protect_from on), the lower
// slot first, then by weight, largest first, the lower slot first among equals.  A weight
// of NaN ranks as the lowest value, +inf below the protected ones.  The kept slots that lie at n or past it move into the slots
// below n that were dropped, the i-th into the i-th: keys carry their rotation, so
// a slot's place does not matter, and nothing else has to move.  Sources lie at n or
// past it and destinations below n, so the moves are independent of one another.
//
// A cluster of 1 to 8 CTAs takes a (sequence, kv head), a stretch of the slots each: the keys
// are read once into shared memory (49152 of them a CTA, in the workspace past that), the
// n-th largest is found from histograms of 11, 11 and 10 bits that the CTAs add up over
// distributed shared memory.  Then each thread walks consecutive slots of its CTA's
// stretch, and block-wide prefix sums, offset by the counts of the CTAs before, number the
// ties, the dropped slots below n and the kept slots past it.  (One CTA a head with the
// keys read again for each of four 8-bit digits and a scan for every 1024 slots took 87 us
// for 32 heads of 30011 slots, with 11-bit digits and one read 36 us; clusters of
// 4 take 22 to 24 us, and the whole eviction to 4096 slots 39 to 42 us.)
#include <cooperative_groups.h>

#include <algorithm>

#include "launch.cuh"
#include "paged.cuh"

namespace w4a8 {

namespace {

constexpr int kSelThreads = 1024;
constexpr int kMoveThreads = 256;
constexpr int kSharedKeys = 49152;  // slots whose keys fit in a CTA's shared memory
constexpr int kMaxCluster = 8;
constexpr int kBins = 2048;

struct EvictParams {
    int KVH, D;
    const float* acc;
    const uint32_t* pos;
    int stride;  // slots of a row of acc and pos, in and out
    const uint32_t* keep;
    const uint32_t* protect_from;
    bool limits_signed;  // keep and protect_from are two's complement, below zero as zero
    int sink;
    float* acc_out;
    uint32_t* pos_out;
    uint32_t* len_out;
    // workspace: per (sequence, kv head) the count of moves, then its destinations and sources
    uint32_t* count;
    uint32_t* moves;  // [batch * KVH][2][stride / 2 + 1]: at most half of the slots move
    uint32_t* keys;   // [batch * KVH][stride], or NULL: in shared memory
    PagedCache c;
    PagedBatch b;
};

// An entry of keep or protect_from.
__device__ __forceinline__ uint32_t limit_of(const EvictParams& p, const uint32_t* at) {
    const uint32_t x = ld_dep(at);
    return p.limits_signed ? static_cast<uint32_t>(max(static_cast<int>(x), 0)) : x;
}

// Slots of a sequence, as far as acc and pos reach, and how many of them stay.
__device__ __forceinline__ int slots_of(const EvictParams& p, int seq) {
    const uint32_t cap = min(static_cast<uint32_t>(p.b.table_stride) * static_cast<uint32_t>(p.c.page),
                             static_cast<uint32_t>(p.stride));
    return static_cast<int>(min(ld_dep(p.b.kv_len + seq), cap));
}
__device__ __forceinline__ int kept_of(const EvictParams& p, int seq, int len) {
    return static_cast<int>(min(static_cast<uint32_t>(len), limit_of(p, p.keep + seq)));
}

// Unsigned key in the order of the ranking: larger stays longer.
__device__ __forceinline__ uint32_t rank_key(float w, uint32_t pos, int sink, uint32_t protect_from) {
    if (pos < static_cast<uint32_t>(sink) || pos >= protect_from) return 0xffffffffu;  // past +inf's key, 0xff800000
    if (w != w) return 0x007fffffu;                                                     // -inf's key
    const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Exclusive prefix sum of v over the CTA; total gets the sum.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* red, uint32_t& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t x = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const uint32_t y = __shfl_up_sync(kFull, x, off);
        if (lane >= off) x += y;
    }
    __syncthreads();
    if (lane == 31) red[warp] = x;
    __syncthreads();
    uint32_t w = red[lane];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const uint32_t y = __shfl_up_sync(kFull, w, off);
        if (lane >= off) w += y;
    }
    total = __shfl_sync(kFull, w, 31);
    const uint32_t before = warp ? __shfl_sync(kFull, w, warp - 1) : 0u;
    return before + x - v;
}

__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictParams p) {
    namespace cg = cooperative_groups;
    extern __shared__ uint32_t shared_keys[];
    __shared__ uint32_t hist[2][kBins];  // by turns, so that a pass may clear one while a neighbour still reads the other
    __shared__ uint32_t red[32];
    __shared__ uint32_t pick[3];
    __shared__ uint32_t counts[3];  // dropped slots below n, kept slots past it, ties
    pdl_launch_dependents();
    pdl_wait();
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
    const int kh = blockIdx.x / ctas, seq = blockIdx.y, tid = threadIdx.x;
    const int len = slots_of(p, seq), n = kept_of(p, seq, len);
    const uint32_t from = limit_of(p, p.protect_from + seq);
    const size_t row = static_cast<size_t>(seq) * p.KVH + kh;
    const float* acc = p.acc + row * p.stride;
    const uint32_t* pos = p.pos + row * p.stride;
    float* acc_out = p.acc_out + row * p.stride;
    uint32_t* pos_out = p.pos_out + row * p.stride;
    // this CTA's slots
    const int part = (len + ctas - 1) / ctas;
    const int s0 = min(rank * part, len), mine = min(part, len - s0);
    if (n == len || n == 0) {  // nothing goes, or everything: the whole cluster leaves here
        if (rank == 0 && tid == 0) p.count[row] = 0;
        if (n > 0 && (acc_out != acc || pos_out != pos))
            for (int j = s0 + tid; j < s0 + mine; j += kSelThreads) {
                acc_out[j] = ld_dep(acc + j);
                pos_out[j] = ld_dep(pos + j);
            }
        return;
    }
    uint32_t* keys = p.keys ? p.keys + row * p.stride + s0 : shared_keys;

    // the n-th largest key: `prefix` down to its known bits, of the slots that match it so far the first `left` stay
    uint32_t prefix = 0, left = static_cast<uint32_t>(n), match = static_cast<uint32_t>(len);
    int low = 32;  // bits below the known ones
    for (int pass = 0; pass < 3 && left < match; ++pass) {
        const int bits = pass == 2 ? 10 : 11, shift = low - bits;
        uint32_t* h = hist[pass & 1];
        for (int b = tid; b < kBins; b += kSelThreads) h[b] = 0;
        __syncthreads();
        auto count = [&](uint32_t key, bool live) {
            const uint32_t bin = (key >> shift) & ((1u << bits) - 1);
            int same;
            __match_all_sync(kFull, live ? bin : ~0u, &same);
            if (same) {  // ties come in runs: one addition for the warp
                if (live && (tid & 31) == 0) atomicAdd(&h[bin], 32u);
            } else if (live) {
                atomicAdd(&h[bin], 1u);
            }
        };
        constexpr int kAhead = 8;
        for (int j0 = 0; j0 < mine; j0 += kSelThreads * kAhead) {
            if (pass == 0) {
                float w[kAhead];
                uint32_t at[kAhead];
#pragma unroll
                for (int x = 0; x < kAhead; ++x) {
                    const int j = j0 + x * kSelThreads + tid;
                    w[x] = j < mine ? ld_dep(acc + s0 + j) : 0.f;
                    at[x] = j < mine ? ld_dep(pos + s0 + j) : 0u;
                }
#pragma unroll
                for (int x = 0; x < kAhead; ++x) {
                    const int j = j0 + x * kSelThreads + tid;
                    if (j0 + x * kSelThreads >= mine) break;
                    const uint32_t key = rank_key(w[x], at[x], p.sink, from);
                    if (j < mine) keys[j] = key;
                    count(key, j < mine);
                }
            } else {
#pragma unroll
                for (int x = 0; x < kAhead; ++x) {
                    const int j = j0 + x * kSelThreads + tid;
                    if (j0 + x * kSelThreads >= mine) break;
                    const uint32_t key = j < mine ? keys[j] : 0u;
                    const bool live = j < mine && (key >> low) == (prefix >> low);
                    if (__any_sync(kFull, live)) count(key, live);
                }
            }
        }
        cluster.sync();
        // from the top bin down: the bin in which the n-th largest lies
        uint32_t total;
        const int top = (1 << bits) - 1 - 2 * tid;  // this thread's two bins: top, top - 1
        uint32_t c0 = 0, c1 = 0;
        if (top > 0)
            for (int q = 0; q < ctas; ++q) {
                const uint32_t* other = cluster.map_shared_rank(h, q);
                c0 += other[top];
                c1 += other[top - 1];
            }
        const uint32_t above = block_scan(c0 + c1, red, total);
        if (above < left && above + c0 >= left) {
            pick[0] = static_cast<uint32_t>(top);
            pick[1] = left - above;
            pick[2] = c0;
        } else if (above + c0 < left && above + c0 + c1 >= left) {
            pick[0] = static_cast<uint32_t>(top - 1);
            pick[1] = left - above - c0;
            pick[2] = c1;
        }
        __syncthreads();
        prefix |= pick[0] << shift;
        left = pick[1];
        match = pick[2];
        low = shift;
    }
    __syncthreads();
    // Kept: keys above the prefix's bits, and of those that match it the first `left` by slot.

    // consecutive slots a thread; an odd number keeps the threads on different banks
    const int run = ((mine + kSelThreads - 1) / kSelThreads) | 1;
    const int b0 = min(tid * run, mine), b1 = min(b0 + run, mine);
    const uint32_t bar = prefix >> low;
    const bool some = left < match;  // not all of the matching slots stay
    // what the CTAs before have of counts[which], after this one's total is in its own
    auto before = [&](int which, uint32_t total) {
        if (tid == 0) counts[which] = total;
        cluster.sync();
        uint32_t sum = 0;
        for (int q = 0; q < rank; ++q) sum += *cluster.map_shared_rank(&counts[which], q);
        return sum;
    };
    uint32_t total, ties = 0;
    if (some) {
        for (int j = b0; j < b1; ++j) ties += (keys[j] >> low) == bar;
        ties = block_scan(ties, red, total);
        ties += before(2, total);
    }
    uint32_t holes = 0, sources = 0;
    for (int j = b0; j < b1; ++j) {
        const uint32_t k = keys[j] >> low;
        bool kept = k > bar;
        if (k == bar) kept = !some || ties++ < left;
        keys[j] = kept;
        holes += s0 + j < n && !kept;
        sources += s0 + j >= n && kept;
    }
    uint32_t source_total;
    uint32_t hole_at = block_scan(holes, red, total);
    uint32_t source_at = block_scan(sources, red, source_total);
    if (tid == 0) {
        counts[0] = total;
        counts[1] = source_total;
    }
    cluster.sync();
    uint32_t all = 0;
    for (int q = 0; q < ctas; ++q) {
        const uint32_t* other = cluster.map_shared_rank(counts, q);
        if (q < rank) {
            hole_at += other[0];
            source_at += other[1];
        }
        all += other[0];
    }
    uint32_t* dst = p.moves + row * 2 * (p.stride / 2 + 1);
    uint32_t* src = dst + p.stride / 2 + 1;
    for (int j = b0; j < b1; ++j) {
        const bool kept = keys[j] != 0;
        if (s0 + j < n && !kept) dst[hole_at++] = static_cast<uint32_t>(s0 + j);
        if (s0 + j >= n && kept) src[source_at++] = static_cast<uint32_t>(s0 + j);
    }
    if (rank == 0 && tid == 0) p.count[row] = all;
    if (acc_out != acc || pos_out != pos)
        for (int j = tid; j < min(mine, n - s0); j += kSelThreads)
            if (keys[j]) {
                acc_out[s0 + j] = ld_dep(acc + s0 + j);
                pos_out[s0 + j] = ld_dep(pos + s0 + j);
            }
    cluster.sync();  // no CTA leaves while a neighbour reads its counts
}

__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int seq = blockIdx.y / p.KVH, kh = blockIdx.y % p.KVH;
    // the new length: here, where no CTA reads the batch's limits any more, so that it may take their place
    if (kh == 0 && blockIdx.x == 0 && threadIdx.x == 0)
        p.len_out[seq] = static_cast<uint32_t>(kept_of(p, seq, slots_of(p, seq)));
    const size_t row = blockIdx.y;
    const uint32_t count = ld_dep(p.count + row);
    const uint32_t* dst = p.moves + row * 2 * (p.stride / 2 + 1);
    const uint32_t* src = dst + p.stride / 2 + 1;
    const int per = p.D / 8;  // 16-byte pieces of a row
    const uint64_t total = static_cast<uint64_t>(count) * per;
    for (uint64_t e = blockIdx.x * kMoveThreads + threadIdx.x; e < total; e += gridDim.x * kMoveThreads) {
        const uint32_t i = static_cast<uint32_t>(e / per);
        const int d = static_cast<int>(e - static_cast<uint64_t>(i) * per) * 8;
        const size_t a = slot_offset(p.b, p.c, seq, kh, static_cast<int>(ld_dep(src + i))) + d;
        const size_t b = slot_offset(p.b, p.c, seq, kh, static_cast<int>(ld_dep(dst + i))) + d;
        if (d == 0) {  // the move's first piece takes the weight and the position along
            const size_t from = row * p.stride + ld_dep(src + i), to = row * p.stride + ld_dep(dst + i);
            p.acc_out[to] = ld_dep(p.acc + from);
            p.pos_out[to] = ld_dep(p.pos + from);
        }
        const uint4 k = ld_dep(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.c.k) + a));
        const uint4 v = ld_dep(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.c.v) + a));
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.c.k) + b) = k;
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.c.v) + b) = v;
    }
}

}  // namespace

int sm_count();  // capi.cu

namespace {

size_t workspace_of(int batch, int KVH, int stride) {
    if (batch < 1 || KVH < 1 || stride < 1) return 0;
    const size_t rows = static_cast<size_t>(batch) * KVH;
    const size_t moves = rows * 2 * (static_cast<size_t>(stride) / 2 + 1) * 4;
    return (rows * 4 + 255) / 256 * 256 + (moves + 255) / 256 * 256 + (stride > kSharedKeys ? rows * stride * 4 : 0);
}

w4a8_status evict(const char* what, bool limits_signed, void* k, void* v, int dtype, int pages, int page, size_t page_stride,
                  int head_stride, int row_stride, int KVH, int D, const uint32_t* kv_len, const uint32_t* table, int batch,
                  int table_stride, const float* acc, const uint32_t* pos, int stride, const uint32_t* keep,
                  const uint32_t* protect_from, int sink, float* acc_out, uint32_t* pos_out, uint32_t* len_out,
                  void* workspace, size_t workspace_bytes, void* stream) {
    EvictParams p{};
    p.limits_signed = limits_signed;
    p.c = PagedCache{k, v, dtype, pages, page, page_stride, head_stride, row_stride};
    // no new tokens here: kv_len stands in for the starts, which no kernel below reads
    p.b = PagedBatch{kv_len, kv_len, table, batch, table_stride, 0};
    w4a8_status st = check_heads(what, KVH, KVH, D);
    if (st == W4A8_OK) st = check_cache(what, p.c, KVH, D);
    if (st == W4A8_OK) st = check_batch(what, p.b);
    if (st != W4A8_OK) return st;
    if (static_cast<long long>(table_stride) * page >= (1ll << 31))
        return set_error(W4A8_EINVAL, "%s: %d pages of %d slots a sequence", what, table_stride, page);
    if (!acc || !pos || !keep || !protect_from || !acc_out || !pos_out || !len_out)
        return set_error(W4A8_EINVAL, "%s: NULL pointer", what);
    if (stride < 1 || sink < 0) return set_error(W4A8_EINVAL, "%s: %d slots a head, sink %d", what, stride, sink);
    if (len_out == kv_len) return set_error(W4A8_EINVAL, "%s: len_out is kv_len", what);
    if (static_cast<long long>(batch) * KVH > 65535)
        return set_error(W4A8_EINVAL, "%s: %d sequences of %d heads (at most 65535 in all)", what, batch, KVH);
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < workspace_of(batch, KVH, stride))
        return set_error(W4A8_EINVAL, "%s: workspace NULL, small or misaligned", what);
    p.KVH = KVH;
    p.D = D;
    p.acc = acc;
    p.pos = pos;
    p.stride = stride;
    p.keep = keep;
    p.protect_from = protect_from;
    p.sink = sink;
    p.acc_out = acc_out;
    p.pos_out = pos_out;
    p.len_out = len_out;
    const size_t rows = static_cast<size_t>(batch) * KVH;
    p.count = static_cast<uint32_t*>(workspace);
    p.moves = p.count + ((rows * 4 + 255) / 256) * 64;
    cudaStream_t cs = static_cast<cudaStream_t>(stream);
    // as many CTAs a head as leave each 2048 slots and find an SM each, up to 8
    int ctas = 1;
    while (ctas < kMaxCluster && rows * ctas * 2 <= static_cast<size_t>(sm_count()) && stride / (ctas * 2) >= 2048) ctas *= 2;
    const int part = (stride + ctas - 1) / ctas;
    p.keys = part > kSharedKeys ? p.moves + (rows * 2 * (static_cast<size_t>(stride) / 2 + 1) + 63) / 64 * 64 : nullptr;
    static FuncAttr attr;
    st = ensure_smem(evict_select_kernel, attr, static_cast<size_t>(kSharedKeys) * 4, -1, what);
    if (st != W4A8_OK) return st;
    const dim3 grid(KVH * ctas, batch);
    const size_t smem = p.keys ? 0 : static_cast<size_t>(part) * 4;
    st = ctas == 1 ? launch_pdl(what, evict_select_kernel, grid, dim3(kSelThreads), smem, cs, p)
                   : launch_cluster(what, evict_select_kernel, grid, dim3(kSelThreads), smem, ctas, cs, p);
    if (st != W4A8_OK) return st;
    // enough CTAs to fill the GPU, no more a head than its most moves take
    const long long most = (static_cast<long long>(stride) / 2 + 1) * (D / 8);
    long long per = (8ll * sm_count() + rows - 1) / static_cast<long long>(rows);
    per = std::min<long long>(per, (most + kMoveThreads - 1) / kMoveThreads);
    return launch_pdl(what, evict_move_kernel, dim3(static_cast<unsigned>(per), static_cast<unsigned>(rows)),
                      dim3(kMoveThreads), 0, cs, p);
}

}  // namespace

}  // namespace w4a8

using namespace w4a8;

extern "C" {

W4A8_API size_t w4a8_kv_evict_workspace_bytes(int32_t batch, int32_t KVH, int32_t stride) {
    return workspace_of(batch, KVH, stride);
}

W4A8_API w4a8_status w4a8_kv_evict(void* k, void* v, int32_t dtype, int32_t pages, int32_t page, size_t page_stride,
                                   int32_t head_stride, int32_t row_stride, int32_t KVH, int32_t D,
                                   const uint32_t* kv_len, const uint32_t* table, int32_t batch, int32_t table_stride,
                                   const float* acc, const uint32_t* pos, int32_t stride, const uint32_t* keep,
                                   const uint32_t* protect_from, int32_t sink, float* acc_out, uint32_t* pos_out,
                                   uint32_t* len_out, void* workspace, size_t workspace_bytes, void* stream) {
    return evict("w4a8_kv_evict", false, k, v, dtype, pages, page, page_stride, head_stride, row_stride, KVH, D, kv_len, table,
                 batch, table_stride, acc, pos, stride, keep, protect_from, sink, acc_out, pos_out, len_out, workspace,
                 workspace_bytes, stream);
}

W4A8_API w4a8_status w4a8_kv_evict_signed(void* k, void* v, int32_t dtype, int32_t pages, int32_t page, size_t page_stride,
                                          int32_t head_stride, int32_t row_stride, int32_t KVH, int32_t D,
                                          const uint32_t* kv_len, const uint32_t* table, int32_t batch,
                                          int32_t table_stride, const float* acc, const uint32_t* pos, int32_t stride,
                                          const uint32_t* keep, const uint32_t* protect_from, int32_t sink, float* acc_out,
                                          uint32_t* pos_out, uint32_t* len_out, void* workspace, size_t workspace_bytes,
                                          void* stream) {
    return evict("w4a8_kv_evict_signed", true, k, v, dtype, pages, page, page_stride, head_stride, row_stride, KVH, D, kv_len,
                 table, batch, table_stride, acc, pos, stride, keep, protect_from, sink, acc_out, pos_out, len_out, workspace,
                 workspace_bytes, stream);
}

}  // extern "C"
