// The attention weight that each cached slot received from the step's new tokens,
// added to what it had:
//
//   acc[b, kvh, j] += sum over new tokens i that see j, query heads h of kvh, of
//                     exp(scale q_ih . k_j - lse_ih)
//
// The sum over rows belongs to one CTA for each slot, in a fixed order: no atomics, and
// the same inputs give the same bits.
#include "launch.cuh"
#include "paged.cuh"

namespace w4a8 {

namespace {

constexpr int kRows = 16, kKeys = 32, kThreads = 128;

struct WeightParams {
    const void* q;
    int q_row, H, KVH, D;
    float scale;
    const float* lse;
    float* acc;
    int acc_stride, max_q;
    PagedCache c;
    PagedBatch b;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) weights_rows_kernel(const WeightParams p) {
    extern __shared__ float sm[];
    pdl_launch_dependents();
    pdl_wait();
    const int G = p.H / p.KVH, D = p.D, ld = D + 1;
    const int seq = blockIdx.z, kh = blockIdx.y, j0 = blockIdx.x * kKeys;
    const SeqSpan sp = seq_span(p.b, p.c, seq);
    const int rows = min(sp.n, p.max_q) * G;
    const int len = min(sp.len, p.acc_stride);
    if (j0 >= len || rows == 0) return;
    float* qs = sm;               // [16][D + 1]
    float* ks = qs + kRows * ld;  // [32][D + 1]
    float* ps = ks + kKeys * ld;  // [16][33]
    const int tid = threadIdx.x;
    for (int e = tid; e < kKeys * D; e += kThreads) {
        const int j = j0 + e / D, d = e % D;
        ks[(e / D) * ld + d] =
            j < len ? static_cast<float>(ld_dep(static_cast<const T*>(p.c.k) + slot_offset(p.b, p.c, seq, kh, j) + d)) : 0.f;
    }
    float total = 0.f;
    for (int r0 = 0; r0 < rows; r0 += kRows) {
        __syncthreads();
        for (int e = tid; e < kRows * D; e += kThreads) {
            const int r = e / D, d = e % D, rr = min(r0 + r, rows - 1);
            const size_t at = static_cast<size_t>(sp.t0 + rr / G) * p.q_row + static_cast<size_t>(kh * G + rr % G) * D + d;
            qs[r * ld + d] = static_cast<float>(ld_dep(static_cast<const T*>(p.q) + at)) * p.scale;
        }
        __syncthreads();
        for (int e = tid; e < kRows * kKeys; e += kThreads) {
            const int r = e / kKeys, j = e % kKeys;
            float w = 0.f;
            if (r0 + r < rows && j0 + j < len && j0 + j <= sp.len - sp.n + (r0 + r) / G) {
                float s = 0.f;
                for (int d = 0; d < D; ++d) s += qs[r * ld + d] * ks[j * ld + d];
                const int t = sp.t0 + (r0 + r) / G, h = kh * G + (r0 + r) % G;
                w = expf(s - ld_dep(p.lse + static_cast<size_t>(t) * p.H + h));
            }
            ps[r * 33 + j] = w;
        }
        __syncthreads();
        if (tid < kKeys) {
            float s = 0.f;
            for (int r = 0; r < kRows; ++r) s += ps[r * 33 + tid];
            total += s;
        }
    }
    if (tid < kKeys && j0 + tid < len)
        p.acc[(static_cast<size_t>(seq) * p.KVH + kh) * p.acc_stride + j0 + tid] += total;
}

}  // namespace
}  // namespace w4a8

using namespace w4a8;

extern "C" {

W4A8_API w4a8_status w4a8_attn_weights(const void* q, int32_t q_row_stride, const float* lse, int32_t H, int32_t KVH,
                                       int32_t D, float scale, const uint32_t* q_start, const uint32_t* kv_len,
                                       const uint32_t* table, int32_t batch, int32_t table_stride, int32_t tokens,
                                       int32_t max_q, int32_t max_kv, const void* k, int32_t dtype, int32_t pages,
                                       int32_t page, size_t page_stride, int32_t head_stride, int32_t row_stride,
                                       float* acc, int32_t acc_stride, void* stream) {
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
    if (!(scale == scale) || scale < 0.f) return set_error(W4A8_EINVAL, "%s: scale %g", what, scale);
    if (tokens == 0 || max_q == 0 || max_kv == 0) return W4A8_OK;
    p.q = q;
    p.q_row = q_row_stride;
    p.H = H;
    p.KVH = KVH;
    p.D = D;
    p.scale = scale;
    p.lse = lse;
    p.acc = acc;
    p.acc_stride = acc_stride;
    p.max_q = max_q;
    const size_t smem = static_cast<size_t>((kRows + kKeys) * (D + 1) + kRows * 33) * 4;
    const dim3 grid((static_cast<unsigned>(max_kv) + kKeys - 1) / kKeys, KVH, batch);
    static FuncAttr a16, ab16;
    cudaStream_t cs = static_cast<cudaStream_t>(stream);
    if (dtype == W4A8_F16) {
        st = ensure_smem(weights_rows_kernel<__half>, a16, smem, -1, what);
        return st != W4A8_OK ? st : launch_pdl(what, weights_rows_kernel<__half>, grid, dim3(kThreads), smem, cs, p);
    }
    st = ensure_smem(weights_rows_kernel<__nv_bfloat16>, ab16, smem, -1, what);
    return st != W4A8_OK ? st : launch_pdl(what, weights_rows_kernel<__nv_bfloat16>, grid, dim3(kThreads), smem, cs, p);
}

}  // extern "C"
