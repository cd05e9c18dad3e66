// tcgen05 helpers for 16-bit operands, of one SM and of pairs, shared by the attention
// kernels: tensor memory, descriptors of 128-byte-swizzled tiles, kind::f16 MMAs, the tensor
// maps of a paged cache and of query rows, places on a work line, and bounded waits.  No load here uses cluster multicast.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "paged.cuh"
#include "tma.cuh"

namespace w4a8 {

unsigned int* device_error_word();  // gemv_mma.cu

__device__ __forceinline__ void tc1_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc1_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tmem1_alloc(uint32_t* slot, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem1_dealloc(uint32_t taddr, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
__device__ __forceinline__ void tmem1_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem1_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 consecutive 32-bit columns of this thread's lane.
__device__ __forceinline__ void tmem1_ld32(uint32_t taddr, float* f) {
    uint32_t* r = reinterpret_cast<uint32_t*>(f);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem1_st32(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
        "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
        "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}

// 16 columns.
__device__ __forceinline__ void tmem1_ld16(uint32_t taddr, float* f) {
    uint32_t* r = reinterpret_cast<uint32_t*>(f);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem1_st16(uint32_t taddr, const uint32_t* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}

// Shared-memory operands in the 128-byte swizzle, tiles of rows of 128 bytes (64
// elements) with 8-row atoms 1024 bytes apart.
// K-major: the row is the M or N index, its bytes run along K; a k-step of 16 elements
// is 32 bytes further.
__device__ __forceinline__ uint64_t desc_k_major(uint32_t saddr) {
    uint64_t d = static_cast<uint64_t>((saddr >> 4) & 0x3FFFu);
    d |= static_cast<uint64_t>(1) << 16;
    d |= static_cast<uint64_t>(1024 >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}
// MN-major: the row is the K index, its bytes run along N; tiles of the next 64 N lie
// `tile` bytes further (leading byte offset), the next 8 K 1024 bytes (stride byte
// offset), so a k-step of 16 is 2048 bytes further.
__device__ __forceinline__ uint64_t desc_mn_major(uint32_t saddr, uint32_t tile) {
    uint64_t d = static_cast<uint64_t>((saddr >> 4) & 0x3FFFu);
    d |= static_cast<uint64_t>(tile >> 4) << 16;
    d |= static_cast<uint64_t>(1024 >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}

// kind::f16 instruction descriptor: f32 accumulator of 128 x n, A and B both f16 or
// both bf16, A K-major, B K-major or MN-major.
template <typename T>
__host__ __device__ constexpr uint32_t idesc_f16(int n, bool b_mn_major) {
    const uint32_t type = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (type << 7) | (type << 10) | ((b_mn_major ? 1u : 0u) << 16) |
           (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(128 >> 4) << 24);
}

__device__ __forceinline__ void mma_f16_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(acc)
        : "memory");
}
// Arrives on the barrier once the MMAs this thread has issued so far complete.
__device__ __forceinline__ void tc1_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
// The same for a pair of CTAs (cta_group::2): M = 256, each CTA's 128 rows of A and D its own,
// half of B's N in each CTA's shared memory.  One thread of CTA 0 issues.
template <typename T>
__host__ __device__ constexpr uint32_t idesc_f16_pair(int n, bool b_mn_major) {
    return (idesc_f16<T>(n, b_mn_major) & 0x00ffffffu) | (static_cast<uint32_t>(256 >> 4) << 24);
}
__device__ __forceinline__ void mma_f16_ss_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_f16_ts_pair(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(acc)
        : "memory");
}
// Arrives on this barrier of both CTAs once the pair's MMAs so far complete (a completion signal, not a load).
__device__ __forceinline__ void tc2_commit_both(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                     smem_u32(bar)),
                 "h"(static_cast<unsigned short>(3))
                 : "memory");
}
__device__ __forceinline__ void tmem2_alloc(uint32_t* slot, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem2_dealloc(uint32_t taddr, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
__device__ __forceinline__ uint32_t pair_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void pair_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Arrival on a barrier of CTA `rank` of the pair, after what this thread has seen and written.
__device__ __forceinline__ void mbar_arrive_at(uint64_t* bar, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(bar)), "r"(rank));
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(r) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void tma_load_3d_at(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}

// The largest of three (one instruction).
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Sum over a warp of lengths on a work line, none negative.  What 32 bits hold (nearly every batch) is one
// reduction; longer ones are summed in 64 bits, cut at 2^40, so that no sum of them wraps.
__device__ __forceinline__ long long line_sum(long long x) {
    if (!__any_sync(kFull, (x >> 25) != 0)) return __reduce_add_sync(kFull, static_cast<unsigned>(x));
    x = min(x, 1ll << 40);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) x += __shfl_xor_sync(kFull, x, off);
    return x;
}
// A sequence's line for all of its kv heads.
__device__ __forceinline__ long long line_heads(long long one, int KVH) { return min(min(one, 1ll << 33) * KVH, 1ll << 40); }
// Length of a whole line as the places on it are counted, in 31 bits: a longer one is not walked at all (its places
// would wrap, and with them the heads and tokens found from them); the device error word says so.
__device__ __forceinline__ int line_length(long long total, unsigned int* err) {
    if (total <= 0x7fffffffll) return static_cast<int>(total);
    if ((threadIdx.x & 31) == 0) atomicOr(err, DEV_ERR_ATTN_LINE);
    return 0;
}

// (a * b - less) / c for places on a work line, which are below 2^31; the product nearly always fits 32 bits, and a 64-bit division is some
// hundreds of clocks that a kernel's start would wait for.
__device__ __forceinline__ int line_mul_div(int a, int b, int c, int less = 0) {
    const unsigned long long x = static_cast<unsigned long long>(a) * static_cast<unsigned>(b) - less;
    return static_cast<int>(x >> 32 ? x / static_cast<unsigned>(c) : static_cast<uint32_t>(x) / static_cast<uint32_t>(c));
}

// Bounded waits of a kernel's roles: one that gives up sets the device error word and
// the CTA's abort flag, and every role then leaves its loop.
struct Bail {
    volatile int* flag;
    unsigned int* err;
    // A wait that looks at the flag only where the barrier is not complete yet: a barrier that
    // mostly is costs one test.
    __device__ __forceinline__ bool ready(uint64_t* bar, uint32_t parity) const {
        return mbar_test(bar, parity) || (!*flag && wait(bar, parity));
    }
    __device__ bool wait(uint64_t* bar, uint32_t parity) const {
        if (mbar_wait(bar, parity)) return true;
        *flag = 1;
        atomicOr(err, DEV_ERR_ATTN_TIMEOUT);
        return false;
    }
};

// Tensor maps (attn_paged.cu).  Rows of a page go into a tile in boxes of
// cache_box_rows(page) rows x 64 elements, the largest power of two that divides
// both the page and the tile's 128 rows; elements past D read as zero.
inline int cache_box_rows(int page) { return page % 128 == 0 ? 128 : page & -page; }
// The map's dimensions after the elements go by stride; order gives their coordinates.
struct CacheOrder {
    int id[3];  // 0: row of the page, 1: kv head, 2: page
    __device__ __forceinline__ int pick(int i, int row, int head, int page) const {
        return id[i] == 0 ? row : id[i] == 1 ? head : page;
    }
};
w4a8_status encode_cache(CUtensorMap* map, CacheOrder* order, const void* base, const PagedCache& c, int KVH, int D,
                         int box_rows, const char* what);
// Query rows of one kv head as (64 elements, G heads, tokens) boxes: row = token * G + head.
w4a8_status encode_queries(CUtensorMap* map, const void* q, int dtype, int H, int D, int row_stride, int tokens, int G,
                           int box_tokens, const char* what);

}  // namespace w4a8
