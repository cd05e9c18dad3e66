// Attention of the new tokens of a batch over the paged cache.
//
//   s = scale q . k,  p = exp(s - max),  o = sum p v / sum p,  lse = max + ln sum p
//
// over the slots that the token sees; o times sigmoid(gate) where a gate is given.
// A row that sees nothing gives o = 0 and lse = -inf.
#include "launch.cuh"
#include "paged.cuh"

namespace w4a8 {

namespace {

constexpr int kRows = 16, kKeys = 32, kThreads = 128;

struct AttnParams {
    const void* q;
    int q_row, H, KVH, D;
    float scale;
    const float* gate;
    int gate_row, gate_head;
    void* o;
    int o_type;
    float* lse;
    int max_q;
    PagedCache c;
    PagedBatch b;
};

__device__ __forceinline__ void store_out(void* o, int type, size_t at, float x) {
    if (type == W4A8_F32)
        static_cast<float*>(o)[at] = x;
    else if (type == W4A8_F16)
        static_cast<__half*>(o)[at] = __float2half_rn(Elem<__half>::sat(x));
    else
        static_cast<__nv_bfloat16*>(o)[at] = __float2bfloat16_rn(x);
}

// One CTA takes 16 rows (new token i, query head of the kv head) of one sequence and
// kv head, and walks the slots 32 at a time with a running maximum and sum.
template <typename T>
__global__ void __launch_bounds__(kThreads) attn_rows_kernel(const AttnParams p) {
    extern __shared__ float sm[];
    pdl_launch_dependents();
    pdl_wait();
    const int G = p.H / p.KVH, D = p.D, ld = D + 1;
    const int seq = blockIdx.z, kh = blockIdx.y;
    const SeqSpan sp = seq_span(p.b, p.c, seq);
    const int rows = min(sp.n, p.max_q) * G;
    const int r0 = blockIdx.x * kRows;
    if (r0 >= rows) return;
    float* qs = sm;                 // [16][D + 1]
    float* ks = qs + kRows * ld;    // [32][D + 1]
    float* vs = ks + kKeys * ld;    // [32][D + 1]
    float* ps = vs + kKeys * ld;    // [16][33]
    float* os = ps + kRows * 33;    // [16][D + 1]
    float* ms = os + kRows * ld;    // [16] max, sum, factor
    float* ls = ms + kRows;
    float* fs = ls + kRows;
    const int tid = threadIdx.x;
    for (int e = tid; e < kRows * D; e += kThreads) {
        const int r = e / D, d = e % D, rr = min(r0 + r, rows - 1);
        const size_t at = static_cast<size_t>(sp.t0 + rr / G) * p.q_row + static_cast<size_t>(kh * G + rr % G) * D + d;
        qs[r * ld + d] = static_cast<float>(ld_dep(static_cast<const T*>(p.q) + at)) * p.scale;
        os[r * ld + d] = 0.f;
    }
    if (tid < kRows) {
        ms[tid] = -INFINITY;
        ls[tid] = 0.f;
    }
    const int last = min(r0 + kRows, rows) - 1;
    const int end = min(max(sp.len - sp.n + last / G + 1, 0), sp.len);
    for (int j0 = 0; j0 < end; j0 += kKeys) {
        __syncthreads();
        for (int e = tid; e < kKeys * D; e += kThreads) {
            const int j = j0 + e / D, d = e % D;
            float kx = 0.f, vx = 0.f;
            if (j < end) {
                const size_t at = slot_offset(p.b, p.c, seq, kh, j) + d;
                kx = static_cast<float>(ld_dep(static_cast<const T*>(p.c.k) + at));
                vx = static_cast<float>(ld_dep(static_cast<const T*>(p.c.v) + at));
            }
            ks[(e / D) * ld + d] = kx;
            vs[(e / D) * ld + d] = vx;
        }
        __syncthreads();
        for (int e = tid; e < kRows * kKeys; e += kThreads) {
            const int r = e / kKeys, j = e % kKeys;
            const int sees = sp.len - sp.n + min(r0 + r, rows - 1) / G;  // last slot the row sees
            float s = -INFINITY;
            if (j0 + j < end && j0 + j <= sees) {
                s = 0.f;
                for (int d = 0; d < D; ++d) s += qs[r * ld + d] * ks[j * ld + d];
            }
            ps[r * 33 + j] = s;
        }
        __syncthreads();
        if (tid < kRows) {
            float m = ms[tid];
            for (int j = 0; j < kKeys; ++j) m = fmaxf(m, ps[tid * 33 + j]);
            const float base = m == -INFINITY ? 0.f : m;
            const float f = expf(ms[tid] - base);
            float l = ls[tid] * f;
            for (int j = 0; j < kKeys; ++j) {
                const float e = expf(ps[tid * 33 + j] - base);
                ps[tid * 33 + j] = e;
                l += e;
            }
            ms[tid] = m;
            ls[tid] = l;
            fs[tid] = f;
        }
        __syncthreads();
        for (int e = tid; e < kRows * D; e += kThreads) {
            const int r = e / D, d = e % D;
            const int sees = sp.len - sp.n + min(r0 + r, rows - 1) / G;
            float a = os[r * ld + d] * fs[r];
            for (int j = 0; j < kKeys && j0 + j <= sees; ++j) a += ps[r * 33 + j] * vs[j * ld + d];
            os[r * ld + d] = a;
        }
    }
    __syncthreads();
    for (int e = tid; e < kRows * D; e += kThreads) {
        const int r = e / D, d = e % D;
        if (r0 + r >= rows) continue;
        const int t = sp.t0 + (r0 + r) / G, h = kh * G + (r0 + r) % G;
        const float l = ls[r];
        float o = l > 0.f ? os[r * ld + d] / l : (l == 0.f ? 0.f : os[r * ld + d]);
        if (p.gate) {
            const float g = ld_dep(p.gate + static_cast<size_t>(t) * p.gate_row + static_cast<size_t>(h) * p.gate_head + d);
            o /= 1.f + expf(-g);
        }
        store_out(p.o, p.o_type, (static_cast<size_t>(t) * p.H + h) * D + d, o);
        if (d == 0 && p.lse) p.lse[static_cast<size_t>(t) * p.H + h] = l == 0.f ? -INFINITY : ms[r] + logf(l);
    }
}

}  // namespace
}  // namespace w4a8

using namespace w4a8;

extern "C" {

W4A8_API size_t w4a8_attn_paged_workspace_bytes(int32_t tokens, int32_t H, int32_t KVH, int32_t D, int32_t batch,
                                                int32_t max_q, int32_t max_kv) {
    (void)tokens, (void)H, (void)KVH, (void)D, (void)batch, (void)max_q, (void)max_kv;
    return 256;
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
    if (!(scale == scale) || scale < 0.f) return set_error(W4A8_EINVAL, "%s: scale %g", what, scale);
    if (!workspace || !aligned(workspace, 16) ||
        workspace_bytes < w4a8_attn_paged_workspace_bytes(tokens, H, KVH, D, batch, max_q, max_kv))
        return set_error(W4A8_EINVAL, "%s: workspace NULL, small or misaligned", what);
    if (tokens == 0 || max_q == 0) return W4A8_OK;
    p.q = q;
    p.q_row = q_row_stride;
    p.H = H;
    p.KVH = KVH;
    p.D = D;
    p.scale = scale;
    p.gate = gate;
    p.gate_row = gate_row_stride;
    p.gate_head = gate_head_stride;
    p.o = o;
    p.o_type = o_type;
    p.lse = lse;
    p.max_q = max_q;
    const size_t smem = static_cast<size_t>((2 * kRows + 2 * kKeys) * (D + 1) + kRows * 33 + 3 * kRows) * 4;
    const dim3 grid((static_cast<unsigned>(max_q) * (H / KVH) + kRows - 1) / kRows, KVH, batch);
    static FuncAttr a16, ab16;
    cudaStream_t cs = static_cast<cudaStream_t>(stream);
    if (dtype == W4A8_F16) {
        st = ensure_smem(attn_rows_kernel<__half>, a16, smem, -1, what);
        return st != W4A8_OK ? st : launch_pdl(what, attn_rows_kernel<__half>, grid, dim3(kThreads), smem, cs, p);
    }
    st = ensure_smem(attn_rows_kernel<__nv_bfloat16>, ab16, smem, -1, what);
    return st != W4A8_OK ? st : launch_pdl(what, attn_rows_kernel<__nv_bfloat16>, grid, dim3(kThreads), smem, cs, p);
}

}  // extern "C"
