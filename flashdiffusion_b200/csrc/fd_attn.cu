// Entry points of softmax attention over key spans (declared in
// include/fd_sm100.h): argument checks and the choice of kernels.
#include <algorithm>
#include <cmath>

#include "fd_attn_tc.cuh"

namespace fd {
namespace attn {

// Spans of a packed batch: each row finds its document by bisection.
__global__ void document_spans_kernel(const int32_t* __restrict__ offsets, int n, const int32_t* __restrict__ prefix,
                                      int64_t rows, int causal, int window, int32_t* __restrict__ first,
                                      int32_t* __restrict__ end) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= rows) return;
    int lo = 0, hi = n;   // the number of documents that end at or before row i
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (offsets[mid + 1] <= i) lo = mid + 1;
        else hi = mid;
    }
    int f = 0, e = 0;
    if (lo < n && offsets[lo] <= i) {
        const int64_t a = offsets[lo], z = offsets[lo + 1];
        int64_t ff = a, ee = causal ? i + 1 : z;
        if (window > 0 && i - window + 1 > ff) ff = i - window + 1;
        if (prefix) {
            const int64_t pe = a + max(prefix[lo], 0);
            if (pe > ee) ee = pe;
        }
        if (ee > z) ee = z;
        if (ff < 0) ff = 0;
        if (ee > rows) ee = rows;
        f = (int)ff;
        e = (int)ee;
    }
    first[i] = f;
    end[i] = e;
}

__global__ void prefix_spans_kernel(const int32_t* __restrict__ prefix, int q_len, int k_len, int32_t* __restrict__ first,
                                    int32_t* __restrict__ end) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x, b = blockIdx.y;
    if (i >= q_len) return;
    const int e = max(k_len - q_len + i + 1, prefix[b]);
    first[(int64_t)b * q_len + i] = 0;
    end[(int64_t)b * q_len + i] = min(max(e, 0), k_len);
}

// A stride that is never taken (extent 1) may be anything: it becomes 0.
static View view(const void* p, const int64_t* s, int batch, int rows, int heads) {
    return {const_cast<void*>(p), batch > 1 ? s[0] : 0, rows > 1 ? s[1] : 0, heads > 1 ? s[2] : 0};
}

// The sizes and switches of a call.  The launches and the workspace query both read them from here, and so cut the
// same work into the same parts.
static Prob sizes_of(const fd_attention_args* r) {
    Prob a{};
    a.first = r->first;
    a.end = r->end;
    a.causal = r->causal != 0;
    // a window that reaches every key is none; this also keeps pos - window inside 32 bits
    a.window = r->window >= (int64_t)r->q_len + r->k_len ? 0 : r->window;
    a.batch = r->batch;
    a.q_len = r->q_len;
    a.k_len = r->k_len;
    a.heads = r->heads;
    a.kv_heads = r->kv_heads;
    a.dim = r->dim;
    a.group = r->kv_heads > 0 ? r->heads / r->kv_heads : 0;
    return a;
}

static int to_prob(const fd_attention_args* r, bool backward, Prob* out) {
    FD_CHECK_ARG(r, "fd_attention: null arguments");
    FD_CHECK_ARG(r->dtype == FD_DTYPE_F32 || r->dtype == FD_DTYPE_F16 || r->dtype == FD_DTYPE_BF16,
                 "fd_attention: dtype %d", r->dtype);
    FD_CHECK_ARG(r->batch >= 0 && r->q_len >= 0 && r->k_len >= 0, "fd_attention: negative size");
    FD_CHECK_ARG(r->q_len <= (1 << 30) && r->k_len <= (1 << 30), "fd_attention: more than 2^30 rows");
    FD_CHECK_ARG(r->dim >= 1 && r->dim <= 256, "fd_attention: dim=%d not in 1..256", r->dim);
    FD_CHECK_ARG(r->heads >= 1 && r->kv_heads >= 1 && r->heads % r->kv_heads == 0,
                 "fd_attention: heads=%d must be a multiple of kv_heads=%d", r->heads, r->kv_heads);
    FD_CHECK_ARG(r->batch <= 65535 && r->heads <= 65535, "fd_attention: batch=%d or heads=%d above 65535", r->batch, r->heads);
    FD_CHECK_ARG(((uintptr_t)r->o_low & 7) == 0, "fd_attention: o_low must be 8-byte aligned");
    // beyond these the constants of a score (scale / cap and the like) leave fp32
    FD_CHECK_ARG(std::abs(r->scale) <= 1e30, "fd_attention: scale=%g must be a number of at most 1e30", r->scale);
    FD_CHECK_ARG(r->cap == 0.0 || (r->cap >= 1e-3 && r->cap <= 1e18), "fd_attention: cap=%g must be 0 or 1e-3 to 1e18", r->cap);
    FD_CHECK_ARG((r->first == nullptr) == (r->end == nullptr), "fd_attention: first and end come together");
    FD_CHECK_ARG(r->window >= 0, "fd_attention: window=%d", r->window);
    FD_CHECK_ARG(!r->first || (!r->causal && !r->window), "fd_attention: spans replace causal and window");
    FD_CHECK_ARG(r->window == 0 || r->causal, "fd_attention: a window needs causal");
    Prob a = sizes_of(r);
    a.q = view(r->q, r->q_stride, r->batch, r->q_len, r->heads);
    a.k = view(r->k, r->k_stride, r->batch, r->k_len, r->kv_heads);
    a.v = view(r->v, r->v_stride, r->batch, r->k_len, r->kv_heads);
    a.o = view(r->o, r->o_stride, r->batch, r->q_len, r->heads);
    a.d_o = view(r->d_o, r->do_stride, r->batch, r->q_len, r->heads);
    a.dq = view(r->dq, r->dq_stride, r->batch, r->q_len, r->heads);
    a.dk = view(r->dk, r->dk_stride, r->batch, r->k_len, r->kv_heads);
    a.dv = view(r->dv, r->dv_stride, r->batch, r->k_len, r->kv_heads);
    a.lse = r->lse;
    a.o_low = r->o_low;
    a.span_stride = r->span_stride;
    a.lengths = r->lengths;
    a.slopes = r->slopes;
    a.scale = (float)r->scale;
    a.cap = (float)r->cap;
    *out = a;
    if (a.batch == 0) return FD_OK;
    FD_CHECK_ARG(a.q_len == 0 || (a.q.p && a.o.p), "fd_attention: null q or o");
    FD_CHECK_ARG(a.k_len == 0 || (a.k.p && a.v.p), "fd_attention: null k or v");
    if (backward) {
        FD_CHECK_ARG(a.q_len == 0 || (a.d_o.p && a.dq.p && a.lse), "fd_attention_backward: null d_o, dq or lse");
        FD_CHECK_ARG(a.k_len == 0 || (a.dk.p && a.dv.p), "fd_attention_backward: null dk or dv");
    }
    return FD_OK;
}

static size_t delta_bytes(const Prob& a) {
    return align256(sizeof(float) * (size_t)a.batch * a.heads * a.q_len);
}

}  // namespace attn
}  // namespace fd

using namespace fd;

extern "C" {

size_t fd_attention_workspace_bytes(const fd_attention_args* r, int backward) {
    if (!r || r->batch < 0 || r->q_len < 0 || r->k_len < 0 || r->heads < 1) return 0;
    const attn::Prob a = attn::sizes_of(r);
    const bool tc = r->dtype != FD_DTYPE_F32 && a.dim >= 1 && a.kv_heads >= 1;
    if (backward) return std::max(attn::delta_bytes(a), tc && a.dim <= 128 ? attn::tc_backward_bytes(a) : 0);
    if (!tc) return 0;
    return attn::rows_applies(a) ? align256(attn::rows_bytes(a.dim)) : attn::tc_forward_bytes(a);
}

int fd_attention_forward(const fd_attention_args* r, void* workspace, size_t workspace_bytes, void* stream) {
    attn::Prob a;
    FD_TRY(attn::to_prob(r, false, &a));
    if (a.batch == 0 || a.q_len == 0) return FD_OK;
    const size_t need = fd_attention_workspace_bytes(r, 0);
    if (workspace_bytes < need)
        return set_error(FD_ERR_WORKSPACE, "fd_attention_forward: workspace %zu bytes, %zu needed", workspace_bytes, need);
    FD_CHECK_ARG(need == 0 || (workspace && ((uintptr_t)workspace & 255) == 0),
                 "fd_attention_forward: workspace must be 256-byte aligned");
    const bool tc = attn::tc_applies(a, r->dtype, false);
    if (tc && attn::rows_applies(a)) return attn::rows_forward(a, r->dtype, workspace, (cudaStream_t)stream);
    if (tc) return attn::tc_forward(a, r->dtype, workspace, (cudaStream_t)stream);
    return attn::simt_forward(a, r->dtype, (cudaStream_t)stream);
}

int fd_attention_backward(const fd_attention_args* r, void* workspace, size_t workspace_bytes, void* stream) {
    attn::Prob a;
    FD_TRY(attn::to_prob(r, true, &a));
    if (a.batch == 0) return FD_OK;
    const size_t need = fd_attention_workspace_bytes(r, 1);
    if (workspace_bytes < need)
        return set_error(FD_ERR_WORKSPACE, "fd_attention_backward: workspace %zu bytes, %zu needed", workspace_bytes, need);
    FD_CHECK_ARG(need == 0 || (workspace && ((uintptr_t)workspace & 255) == 0),
                 "fd_attention_backward: workspace must be 256-byte aligned");
    if (attn::tc_applies(a, r->dtype, true)) return attn::tc_backward(a, r->dtype, workspace, (cudaStream_t)stream);
    if (!attn::tc_applies(a, r->dtype, false)) a.o_low = nullptr;   // the forward pass was not the one that writes it
    return attn::simt_backward(a, r->dtype, (float*)workspace, (cudaStream_t)stream);
}

int fd_attention_document_spans(const int32_t* offsets, int n_documents, const int32_t* prefix, int64_t rows,
                                int causal, int window, int32_t* first, int32_t* end, void* stream) {
    FD_CHECK_ARG(n_documents >= 0 && rows >= 0 && rows <= (1 << 30), "fd_attention_document_spans: documents=%d rows=%lld",
                 n_documents, (long long)rows);
    FD_CHECK_ARG(window >= 0 && (window == 0 || causal), "fd_attention_document_spans: a window needs causal");
    FD_CHECK_ARG(!prefix || (causal && !window), "fd_attention_document_spans: a prefix needs causal and no window");
    if (rows == 0) return FD_OK;
    FD_CHECK_ARG(offsets && first && end, "fd_attention_document_spans: null pointer");
    attn::document_spans_kernel<<<(unsigned)cdiv(rows, 256), 256, 0, (cudaStream_t)stream>>>(
        offsets, n_documents, prefix, rows, causal, window, first, end);
    FD_CUDA_TRY(cudaGetLastError());
    return FD_OK;
}

int fd_attention_prefix_spans(const int32_t* prefix, int batch, int q_len, int k_len, int32_t* first, int32_t* end,
                              void* stream) {
    FD_CHECK_ARG(batch >= 0 && batch <= 65535 && q_len >= 0 && k_len >= 0 && q_len <= (1 << 30) && k_len <= (1 << 30),
                 "fd_attention_prefix_spans: batch=%d q_len=%d k_len=%d", batch, q_len, k_len);
    if (batch == 0 || q_len == 0) return FD_OK;
    FD_CHECK_ARG(prefix && first && end, "fd_attention_prefix_spans: null pointer");
    attn::prefix_spans_kernel<<<dim3((unsigned)cdiv(q_len, 256), (unsigned)batch), 256, 0, (cudaStream_t)stream>>>(
        prefix, q_len, k_len, first, end);
    FD_CUDA_TRY(cudaGetLastError());
    return FD_OK;
}

}  // extern "C"
