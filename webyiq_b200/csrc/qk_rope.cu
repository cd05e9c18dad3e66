// Norms of queries and keys per head, the position rotation and the append of keys
// and values to the paged cache, in one pass over the projection's rows.
//
//   y = x / sqrt(mean(x^2) + eps) * w            (per head, skipped where w is NULL)
//   (a, b) -> (a cos - b sin, b cos + a sin)     (the first `rot` dims, in pairs)
//   q -> q_out, k and v -> the token's slot
//
// Bound by HBM: 4 bytes read and 2 written for each element, each once.  A group of
// D / 8 lanes (rounded up to 8, 16 or 32) takes one head's row, eight elements a lane
// (two 16-byte loads), so the mean is a few shuffles.  A warp keeps its head (the norm
// weights stay in registers, no division finds a row) and walks the tokens with the next
// row's loads under way.  Measured: 8000 tokens of 32 / 8 heads of 128 in 39.6 us, 4.97 TB/s
// (0.76 of the measured copy rate; 52 us with a row a lane group found by division and
// pairs fetched by shuffles: 60% of the issue slots went to instructions).
#include <algorithm>

#include "launch.cuh"
#include "paged.cuh"

namespace w4a8 {

namespace {

constexpr int kRopeThreads = 256;
constexpr int kBlocksPerSm = 12;

__device__ __forceinline__ float4 ldg4(const float* p) { return __ldg(reinterpret_cast<const float4*>(p)); }

struct RopeParams {
    const float* qkv;
    int row_stride, q_head_stride, H, KVH, D;
    const float* q_norm;
    const float* k_norm;
    float eps;
    const float* rope;
    int rot, rope_rows;
    const uint32_t* pos;
    void* q_out;
    PagedCache c;
    PagedBatch b;
};

// Sequence of new token t: the number of sequences that end at or before it.  A warp
// reads 32 ends at a time, so a batch of up to 32 costs one round trip.
__device__ __forceinline__ int seq_of_token(const PagedBatch& b, int t, int lane) {
    int seq = 0;
    for (int i0 = 0; i0 < b.batch; i0 += 32) {
        const int i = i0 + lane;
        const bool before = i < b.batch && ld_dep(b.q_start + i + 1) <= static_cast<uint32_t>(t);
        const unsigned m = __ballot_sync(kFull, before);
        seq += __popc(m);
        if (m != kFull) break;
    }
    return min(seq, b.batch - 1);
}

template <typename T, int GS, bool EVEN>
__global__ void __launch_bounds__(kRopeThreads) qk_rope_kernel(const RopeParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int heads = p.H + 2 * p.KVH;
    const int gl = lane % GS, e0 = gl * 8;
    // this group's head, the same for every token
    const int h = (blockIdx.y * (kRopeThreads / 32) + (threadIdx.x >> 5)) * (32 / GS) + lane / GS;
    const bool live = h < heads && e0 < p.D, is_q = h < p.H, is_v = h >= p.H + p.KVH;
    const bool stores = __any_sync(kFull, h < heads && !is_q);
    if (!__any_sync(kFull, live)) return;
    // This lane's elements: o0 .. + 3 and o1 .. + 3.  For the pairs (i, i + rot / 2) the second four are the
    // partners of the first, so a rotation needs no shuffle and four angles serve eight elements.
    const int half = p.rot / 2;
    const bool turn = !is_v && live && e0 < p.rot;
    const bool split = !EVEN && e0 < p.rot;
    const int o0 = split ? gl * 4 : e0, o1 = split ? half + gl * 4 : e0 + 4;
    const float* src = p.qkv + (is_q ? static_cast<size_t>(h) * p.q_head_stride
                                          : static_cast<size_t>(p.H) * p.q_head_stride + static_cast<size_t>(h - p.H) * p.D);
    const float* w = is_q ? p.q_norm : p.k_norm;
    const bool normed = !is_v && w && live;
    const float4 w0 = normed ? ldg4(w + o0) : make_float4(1.f, 1.f, 1.f, 1.f);
    const float4 w1 = normed ? ldg4(w + o1) : w0;
    const float inv_d = 1.f / static_cast<float>(p.D);
    auto load = [&](int t, float4& a, float4& b) {
        const float* at = src + static_cast<size_t>(t) * p.row_stride;
        const bool ok = live && t < p.b.tokens;
        a = ok ? ld_dep(reinterpret_cast<const float4*>(at + o0)) : make_float4(0.f, 0.f, 0.f, 0.f);
        b = ok ? ld_dep(reinterpret_cast<const float4*>(at + o1)) : a;
    };
    float4 a, b;
    load(blockIdx.x, a, b);
    for (int t = blockIdx.x; t < p.b.tokens; t += gridDim.x) {
        float y[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        load(t + gridDim.x, a, b);  // the next token's row is under way meanwhile
        // where the row goes: q_out, or the token's slot (none where the sequence is shorter than its new
        // tokens, or the token is none of a sequence's)
        T* dst = is_q ? static_cast<T*>(p.q_out) + (static_cast<size_t>(t) * p.H + h) * p.D : nullptr;
        if (stores) {
            const int seq = seq_of_token(p.b, t, lane);
            const SeqSpan s = seq_span(p.b, p.c, seq);
            const int slot = s.len - s.n + (t - s.t0);
            if (!is_q && h < heads && t >= s.t0 && t < s.t0 + s.n && slot >= 0)
                dst = static_cast<T*>(is_v ? p.c.v : p.c.k) +
                      slot_offset(p.b, p.c, seq, h - p.H - (is_v ? p.KVH : 0), slot);
        }
        float4 c = make_float4(1.f, 1.f, 1.f, 1.f), s = make_float4(0.f, 0.f, 0.f, 0.f);
        if (turn) {  // a row of the table: rot / 2 cosines, then the sines; four angles a lane
            const uint32_t row = min(ld_dep(p.pos + t), static_cast<uint32_t>(p.rope_rows - 1));
            const float* cs = p.rope + static_cast<size_t>(row) * p.rot + gl * 4;
            c = ldg4(cs);
            s = ldg4(cs + half);
        }
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += y[i] * y[i];
#pragma unroll
        for (int off = GS / 2; off > 0; off >>= 1) ss += __shfl_xor_sync(kFull, ss, off);
        const float r = normed ? rsqrtf(ss * inv_d + p.eps) : 1.f;
        y[0] *= r * w0.x;
        y[1] *= r * w0.y;
        y[2] *= r * w0.z;
        y[3] *= r * w0.w;
        y[4] *= r * w1.x;
        y[5] *= r * w1.y;
        y[6] *= r * w1.z;
        y[7] *= r * w1.w;
        const float cc[4] = {c.x, c.y, c.z, c.w}, sc[4] = {s.x, s.y, s.z, s.w};
        if (turn) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float& u = y[EVEN ? 2 * i : i];
                float& v = y[EVEN ? 2 * i + 1 : i + 4];
                const float x0 = u;
                u = x0 * cc[i] - v * sc[i];
                v = v * cc[i] + x0 * sc[i];
            }
        }
        uint2 lo, hi;
        lo.x = Elem<T>::pack(Elem<T>::sat(y[0]), Elem<T>::sat(y[1]));
        lo.y = Elem<T>::pack(Elem<T>::sat(y[2]), Elem<T>::sat(y[3]));
        hi.x = Elem<T>::pack(Elem<T>::sat(y[4]), Elem<T>::sat(y[5]));
        hi.y = Elem<T>::pack(Elem<T>::sat(y[6]), Elem<T>::sat(y[7]));
        if (live && dst) {
            *reinterpret_cast<uint2*>(dst + o0) = lo;
            *reinterpret_cast<uint2*>(dst + o1) = hi;
        }
    }
}

template <typename T, int GS>
w4a8_status launch_rope(const RopeParams& p, bool even, dim3 grid, cudaStream_t st) {
    const char* what = "w4a8_qk_norm_rope_kv";
    return even ? launch_pdl(what, qk_rope_kernel<T, GS, true>, grid, dim3(kRopeThreads), 0, st, p)
                : launch_pdl(what, qk_rope_kernel<T, GS, false>, grid, dim3(kRopeThreads), 0, st, p);
}

}  // namespace

int sm_count();  // capi.cu

w4a8_status check_heads(const char* what, int H, int KVH, int D) {
    if (H < 1 || KVH < 1 || H % KVH || H / KVH > 128)
        return set_error(W4A8_EINVAL, "%s: H=%d KVH=%d (query heads a multiple of the kv heads, at most 128 per kv head)",
                         what, H, KVH);
    if (D < 16 || D > kMaxHeadDim || D % 16)
        return set_error(W4A8_EINVAL, "%s: head dim %d (a multiple of 16, at most %d)", what, D, kMaxHeadDim);
    return W4A8_OK;
}

w4a8_status check_cache(const char* what, const PagedCache& c, int KVH, int D) {
    if (!c.k || !c.v) return set_error(W4A8_EINVAL, "%s: NULL cache", what);
    if (c.dtype != W4A8_F16 && c.dtype != W4A8_BF16)
        return set_error(W4A8_EINVAL, "%s: cache type %d (W4A8_F16 or W4A8_BF16)", what, c.dtype);
    if (!aligned(c.k, 16) || !aligned(c.v, 16)) return set_error(W4A8_EINVAL, "%s: cache not 16-byte aligned", what);
    if (c.pages < 1 || c.page < 16 || c.page > 1024 || c.page % 16)
        return set_error(W4A8_EINVAL, "%s: %d pages of %d slots (a multiple of 16, at most 1024)", what, c.pages, c.page);
    // nested layouts: taken from the smallest stride up, each dimension steps over the ones inside it, so no two
    // elements share an address (a dimension of one has no stride to check)
    struct Dim {
        long long count, stride;
    } d[3] = {{c.page, c.row_stride}, {KVH, c.head_stride}, {c.pages, static_cast<long long>(c.page_stride)}};
    if (c.page_stride >> 38) return set_error(W4A8_EINVAL, "%s: page stride %zu", what, c.page_stride);
    std::sort(d, d + 3, [](const Dim& x, const Dim& y) { return x.stride < y.stride; });
    long long extent = D;
    for (const Dim& x : d) {
        if (x.count == 1) continue;
        if (x.stride < extent || x.stride % 8)
            return set_error(W4A8_EINVAL, "%s: cache strides %zu, %d, %d (multiples of 8 elements, nothing overlapping)",
                             what, c.page_stride, c.head_stride, c.row_stride);
        extent += (x.count - 1) * x.stride;
    }
    return W4A8_OK;
}

w4a8_status check_batch(const char* what, const PagedBatch& b) {
    if (!b.q_start || !b.kv_len || !b.table) return set_error(W4A8_EINVAL, "%s: NULL batch array", what);
    if (b.batch < 1 || b.batch > 65535) return set_error(W4A8_EINVAL, "%s: batch %d (1 to 65535)", what, b.batch);
    if (b.table_stride < 1 || b.table_stride > (1 << 20))
        return set_error(W4A8_EINVAL, "%s: table of %d pages a sequence", what, b.table_stride);
    if (b.tokens < 0 || b.tokens > (1 << 24)) return set_error(W4A8_EINVAL, "%s: tokens %d", what, b.tokens);
    return W4A8_OK;
}

}  // namespace w4a8

using namespace w4a8;

extern "C" {

W4A8_API w4a8_status w4a8_qk_norm_rope_kv(const float* qkv, int32_t row_stride, int32_t q_head_stride, int32_t H,
                                          int32_t KVH, int32_t D, const float* q_norm, const float* k_norm, float eps,
                                          const float* rope, int32_t rot, int32_t rope_rows, int32_t interleaved,
                                          const uint32_t* pos, const uint32_t* q_start, const uint32_t* kv_len,
                                          const uint32_t* table, int32_t batch, int32_t table_stride, int32_t tokens,
                                          void* q_out, void* k, void* v, int32_t dtype, int32_t pages, int32_t page,
                                          size_t page_stride, int32_t head_stride, int32_t row_stride_kv, void* stream) {
    const char* what = "w4a8_qk_norm_rope_kv";
    RopeParams p{};
    p.c = PagedCache{k, v, dtype, pages, page, page_stride, head_stride, row_stride_kv};
    p.b = PagedBatch{q_start, kv_len, table, batch, table_stride, tokens};
    w4a8_status st = check_heads(what, H, KVH, D);
    if (st == W4A8_OK) st = check_cache(what, p.c, KVH, D);
    if (st == W4A8_OK) st = check_batch(what, p.b);
    if (st != W4A8_OK) return st;
    if (static_cast<long long>(table_stride) * page >= (1ll << 31))
        return set_error(W4A8_EINVAL, "%s: %d pages of %d slots a sequence", what, table_stride, page);
    if (tokens > 0 && (!qkv || !q_out || (rot > 0 && (!rope || !pos)))) return set_error(W4A8_EINVAL, "%s: NULL pointer", what);
    if (!aligned(qkv, 16) || !aligned(q_out, 16) || !aligned(q_norm, 16) || !aligned(k_norm, 16) || !aligned(rope, 16))
        return set_error(W4A8_EINVAL, "%s: qkv, q_out, q_norm, k_norm and rope must be 16-byte aligned", what);
    if (q_head_stride < D || q_head_stride % 4 || row_stride % 4 ||
        static_cast<long long>(row_stride) < static_cast<long long>(H) * q_head_stride + 2ll * KVH * D)
        return set_error(W4A8_EINVAL, "%s: row stride %d, query head stride %d (multiples of 4 that hold the heads)", what,
                         row_stride, q_head_stride);
    if (rot < 0 || rot > D || rot % 16 || (rot > 0 && rope_rows < 1))
        return set_error(W4A8_EINVAL, "%s: rotation of %d dims, %d rows (a multiple of 16 up to D)", what, rot, rope_rows);
    if (tokens == 0) return W4A8_OK;
    p.qkv = qkv;
    p.row_stride = row_stride;
    p.q_head_stride = q_head_stride;
    p.H = H;
    p.KVH = KVH;
    p.D = D;
    p.q_norm = q_norm;
    p.k_norm = k_norm;
    p.eps = eps;
    // no rotation: position 0 of any row, never read
    p.rope = rope;
    p.rot = rot;
    p.rope_rows = rot > 0 ? rope_rows : 1;
    p.pos = pos;
    p.q_out = q_out;
    const int gs = D <= 64 ? 8 : D <= 128 ? 16 : 32;
    // a warp keeps its head(s) and walks the tokens; about twelve blocks an SM
    const int per_block = kRopeThreads / gs;
    const int rows = (H + 2 * KVH + per_block - 1) / per_block;
    if (rows > 65535) return set_error(W4A8_EINVAL, "%s: H=%d KVH=%d", what, H, KVH);
    const int wide = std::max(1, sm_count() * kBlocksPerSm / rows);
    const dim3 grid(static_cast<unsigned>(std::min(tokens, wide)), static_cast<unsigned>(rows));
    cudaStream_t cs = static_cast<cudaStream_t>(stream);
    const bool even = interleaved != 0;
    if (dtype == W4A8_F16)
        return gs == 8 ? launch_rope<__half, 8>(p, even, grid, cs)
                       : gs == 16 ? launch_rope<__half, 16>(p, even, grid, cs) : launch_rope<__half, 32>(p, even, grid, cs);
    return gs == 8 ? launch_rope<__nv_bfloat16, 8>(p, even, grid, cs)
                   : gs == 16 ? launch_rope<__nv_bfloat16, 16>(p, even, grid, cs)
                              : launch_rope<__nv_bfloat16, 32>(p, even, grid, cs);
}

}  // extern "C"
