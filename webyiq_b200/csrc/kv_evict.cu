// Eviction from the paged cache by accumulated attention weight.
//
// Per sequence and kv head, of `len` slots the n = min(len, keep) first of this order
// stay: the protected ones (position below `sink`, or from protect_from on), then by
// weight, largest first, the lower slot first among equals.  A weight of NaN ranks
// as the lowest value.  The kept slots that lie at n or past it move into the slots
// below n that were dropped, the i-th into the i-th: keys carry their rotation, so
// a slot's place does not matter, and nothing else has to move.  Sources lie at n or
// past it and destinations below n, so the moves are independent of one another.
//
// The n-th largest key is found digit by digit from histograms; one pass over the
// slots then gives every dropped slot below n and every kept slot past it its number
// by a block-wide prefix sum.
#include <algorithm>

#include "launch.cuh"
#include "paged.cuh"

namespace w4a8 {

namespace {

constexpr int kSelThreads = 1024;
constexpr int kMoveThreads = 256;

struct EvictParams {
    int KVH, D;
    const float* acc;
    const uint32_t* pos;
    int stride;  // slots of a row of acc and pos, in and out
    const uint32_t* keep;
    const uint32_t* protect_from;
    int sink;
    float* acc_out;
    uint32_t* pos_out;
    uint32_t* len_out;
    // workspace: per (sequence, kv head) the count of moves, then its destinations and sources
    uint32_t* count;
    uint32_t* moves;  // [batch * KVH][2][stride]
    PagedCache c;
    PagedBatch b;
};

// Unsigned key in the order of the ranking: larger stays longer.
__device__ __forceinline__ uint32_t rank_key(float w, uint32_t pos, int sink, uint32_t protect_from) {
    if (pos < static_cast<uint32_t>(sink) || pos >= protect_from) return 0xff800000u;  // +inf's key
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
    __shared__ uint32_t hist[256];
    __shared__ uint32_t red[32];
    __shared__ uint32_t pick[2];
    pdl_launch_dependents();
    pdl_wait();
    const int kh = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x;
    const uint32_t cap = min(static_cast<uint32_t>(p.b.table_stride) * static_cast<uint32_t>(p.c.page),
                             static_cast<uint32_t>(p.stride));
    const int len = static_cast<int>(min(ld_dep(p.b.kv_len + seq), cap));
    const int n = static_cast<int>(min(static_cast<uint32_t>(len), ld_dep(p.keep + seq)));
    const uint32_t from = ld_dep(p.protect_from + seq);
    const size_t row = static_cast<size_t>(seq) * p.KVH + kh;
    const float* acc = p.acc + row * p.stride;
    const uint32_t* pos = p.pos + row * p.stride;
    if (kh == 0 && tid == 0) p.len_out[seq] = static_cast<uint32_t>(n);

    // the n-th largest key, and how many slots with that key stay
    uint32_t prefix = 0, left = static_cast<uint32_t>(n);
    for (int shift = 24; shift >= 0 && n > 0 && n < len; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int j = tid; j < len; j += kSelThreads) {
            const uint32_t key = rank_key(ld_dep(acc + j), ld_dep(pos + j), p.sink, from);
            if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(key >> shift) & 255], 1u);
        }
        __syncthreads();
        // slots in larger digits, by a scan from the top digit down
        uint32_t total;
        const uint32_t mine = tid < 256 ? hist[255 - tid] : 0u;
        const uint32_t above = block_scan(mine, red, total);
        if (tid < 256 && above < left && above + mine >= left) {
            pick[0] = static_cast<uint32_t>(255 - tid);
            pick[1] = left - above;
        }
        __syncthreads();
        prefix |= pick[0] << shift;
        left = pick[1];
    }

    uint32_t* dst = p.moves + row * 2 * p.stride;
    uint32_t* src = dst + p.stride;
    uint32_t equal = 0, holes = 0, sources = 0;  // so far
    for (int j0 = 0; j0 < len; j0 += kSelThreads) {
        const int j = j0 + tid;
        bool kept = j < len && n == len;
        if (n < len) {
            uint32_t key = 0;
            if (j < len) key = rank_key(ld_dep(acc + j), ld_dep(pos + j), p.sink, from);
            const bool eq = j < len && n > 0 && key == prefix;
            uint32_t total;
            const uint32_t nth = block_scan(eq ? 1u : 0u, red, total);
            kept = j < len && n > 0 && (key > prefix || (eq && equal + nth < left));
            equal += total;
        }
        const bool hole = j < n && !kept, source = j >= n && kept;
        // both numbers in one scan: at most 1024 of either in a block
        uint32_t total;
        const uint32_t nth = block_scan((hole ? 1u : 0u) | (source ? 1u << 16 : 0u), red, total);
        if (hole) dst[holes + (nth & 0xffffu)] = static_cast<uint32_t>(j);
        if (source) src[sources + (nth >> 16)] = static_cast<uint32_t>(j);
        holes += total & 0xffffu;
        sources += total >> 16;
        if (kept && j < n) {
            p.acc_out[row * p.stride + j] = ld_dep(acc + j);
            p.pos_out[row * p.stride + j] = ld_dep(pos + j);
        }
    }
    __syncthreads();
    for (uint32_t i = tid; i < holes; i += kSelThreads) {
        const uint32_t d = dst[i], s = src[i];
        p.acc_out[row * p.stride + d] = ld_dep(acc + s);
        p.pos_out[row * p.stride + d] = ld_dep(pos + s);
    }
    if (tid == 0) p.count[row] = holes;
}

__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int seq = blockIdx.y / p.KVH, kh = blockIdx.y % p.KVH;
    const size_t row = blockIdx.y;
    const uint32_t count = ld_dep(p.count + row);
    const uint32_t* dst = p.moves + row * 2 * p.stride;
    const uint32_t* src = dst + p.stride;
    const int per = p.D / 8;  // 16-byte pieces of a row
    const uint64_t total = static_cast<uint64_t>(count) * per;
    for (uint64_t e = blockIdx.x * kMoveThreads + threadIdx.x; e < total; e += gridDim.x * kMoveThreads) {
        const uint32_t i = static_cast<uint32_t>(e / per);
        const int d = static_cast<int>(e - static_cast<uint64_t>(i) * per) * 8;
        const size_t a = slot_offset(p.b, p.c, seq, kh, static_cast<int>(ld_dep(src + i))) + d;
        const size_t b = slot_offset(p.b, p.c, seq, kh, static_cast<int>(ld_dep(dst + i))) + d;
        const uint4 k = ld_dep(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.c.k) + a));
        const uint4 v = ld_dep(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.c.v) + a));
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.c.k) + b) = k;
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.c.v) + b) = v;
    }
}

}  // namespace

int sm_count();  // capi.cu

}  // namespace w4a8

using namespace w4a8;

extern "C" {

W4A8_API size_t w4a8_kv_evict_workspace_bytes(int32_t batch, int32_t KVH, int32_t stride) {
    if (batch < 1 || KVH < 1 || stride < 1) return 0;
    const size_t rows = static_cast<size_t>(batch) * KVH;
    return ((rows * 4 + 255) / 256) * 256 + rows * 2 * static_cast<size_t>(stride) * 4;
}

W4A8_API w4a8_status w4a8_kv_evict(void* k, void* v, int32_t dtype, int32_t pages, int32_t page, size_t page_stride,
                                   int32_t head_stride, int32_t row_stride, int32_t KVH, int32_t D,
                                   const uint32_t* kv_len, const uint32_t* table, int32_t batch, int32_t table_stride,
                                   const float* acc, const uint32_t* pos, int32_t stride, const uint32_t* keep,
                                   const uint32_t* protect_from, int32_t sink, float* acc_out, uint32_t* pos_out,
                                   uint32_t* len_out, void* workspace, size_t workspace_bytes, void* stream) {
    const char* what = "w4a8_kv_evict";
    EvictParams p{};
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
    if (len_out == kv_len) return set_error(W4A8_EINVAL, "%s: len_out is kv_len (each head's CTA reads it)", what);
    if (static_cast<long long>(batch) * KVH > 65535)
        return set_error(W4A8_EINVAL, "%s: %d sequences of %d heads (at most 65535 in all)", what, batch, KVH);
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < w4a8_kv_evict_workspace_bytes(batch, KVH, stride))
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
    st = launch_pdl(what, evict_select_kernel, dim3(KVH, batch), dim3(kSelThreads), 0, cs, p);
    if (st != W4A8_OK) return st;
    // enough CTAs to fill the GPU, no more a head than its most moves take
    const long long most = (static_cast<long long>(stride) / 2 + 1) * (D / 8);
    long long per = (8ll * sm_count() + rows - 1) / static_cast<long long>(rows);
    per = std::min<long long>(per, (most + kMoveThreads - 1) / kMoveThreads);
    return launch_pdl(what, evict_move_kernel, dim3(static_cast<unsigned>(per), static_cast<unsigned>(rows)),
                      dim3(kMoveThreads), 0, cs, p);
}

}  // extern "C"
