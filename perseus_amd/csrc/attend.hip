// Attention of packed sequences over keys and values that lie packed or in caches (pcx_attention).
//
// For a query q that sees the keys j: z_j = scale q . k_j, m = max z_j, l = sum exp(z_j - m), o = sum exp(z_j - m) v_j / l,
// lse = m + log l. One pass over the keys holds (m, l, o) and rescales l and o where m grows. Sums, maxima and o are f32.
#include "clear.h"

namespace pch {
namespace clear {

constexpr int BX = 256;
constexpr int DMAX = 256;
constexpr int64_t TOKEN_MAX = 1 << 22;  // key rows' distance, in elements: a tile's byte offsets stay in 32 bits

__device__ __forceinline__ float wg_max(float x, float* sh) {
    for (int m = 32; m; m >>= 1) x = fmaxf(x, __shfl_xor(x, m));
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = x;
    __syncthreads();
    x = fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3]));
    __syncthreads();
    return x;
}
__device__ __forceinline__ float wg_sum(float x, float* sh) {
    for (int m = 32; m; m >>= 1) x += __shfl_xor(x, m);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = x;
    __syncthreads();
    x = sh[0] + sh[1] + sh[2] + sh[3];
    __syncthreads();
    return x;
}

// a workgroup per query and head, a thread per key of each 256, then a thread per output dimension
template <class T>
__global__ void __launch_bounds__(BX) attend_k(AttentionArgs A) {
    __shared__ float q[DMAX], p[BX], sh[4];
    const int t = blockIdx.x, h = blockIdx.y, i = threadIdx.x;
    int b = 0;  // the sequence of row t: the last whose start is not above it
    for (int lo = 0, hi = A.seqs; lo < hi;) {
        const int mid = (lo + hi) >> 1;
        if (A.q_start[mid + 1] > t) hi = mid, b = mid;
        else lo = mid + 1, b = lo;
    }
    if (b >= A.seqs || A.q_start[b] > t) return;
    const int q0 = max(A.q_start[b], 0), n = min(A.q_start[b + 1], A.tokens) - q0;
    int64_t k0 = A.k_start[b], len = A.k_len[b];
    if (k0 < 0 || k0 > A.kv_rows) k0 = len = 0;
    len = max((int64_t)0, min(len, A.kv_rows - k0));
    const int kh = h / (A.heads / A.kv_heads);
    const int64_t seen = A.causal ? min(len, max((int64_t)0, len - n + (t - q0) + 1)) : len;
    if (i < A.dim) q[i] = (float)at<T>(A.q, t, h)[i] * A.scale;
    __syncthreads();
    float m = -INFINITY, l = 0, o = 0;
    for (int64_t j0 = 0; j0 < seen; j0 += BX) {
        float z = -INFINITY;
        if (j0 + i < seen) {
            const T* k = at<T>(A.k, k0 + j0 + i, kh);
            z = 0;
            for (int d = 0; d < A.dim; ++d) z = fmaf(q[d], (float)k[d], z);
        }
        const float mn = fmaxf(m, wg_max(z, sh));
        const float e = j0 + i < seen ? expf(z - mn) : 0.0f, r = m == mn ? 1.0f : expf(m - mn);
        p[i] = e;
        l = l * r + wg_sum(e, sh);
        m = mn;
        if (i < A.dim) {
            o *= r;
            const int c = (int)min((int64_t)BX, seen - j0);
            for (int j = 0; j < c; ++j) o = fmaf(p[j], (float)at<T>(A.v, k0 + j0 + j, kh)[i], o);
        }
        __syncthreads();
    }
    if (i < A.dim) at<T>(A.out, t, h)[i] = (T)(seen > 0 ? o / l : 0.0f);
    if (i == 0 && A.lse) A.lse[(int64_t)t * A.heads + h] = seen > 0 ? m + logf(l) : -INFINITY;
}

// 0, or the error
static int checked(const AttentionArgs* a) {
    if (!a || a->tokens < 0 || a->seqs < 0 || a->heads < 0 || a->kv_heads < 0 || a->kv_rows < 0 || a->max_q < 0 ||
        a->max_k < 0)
        return -1;
    if (a->type != PCX_BF16 && a->type != PCX_F16) return -2;
    if (a->dim < 8 || a->dim > DMAX || a->dim % 8) return -2;
    if (!(a->scale > 0) || a->scale > 3e38f) return -1;
    if (a->heads && (a->kv_heads < 1 || a->heads % a->kv_heads)) return -1;
    if (a->seqs && a->tokens && a->heads && (!a->q_start || !a->k_start || !a->k_len)) return -1;
    if (!usable(a->q, a->tokens, a->heads) || !usable(a->out, a->tokens, a->heads) ||
        !usable(a->k, a->kv_rows, a->kv_heads) || !usable(a->v, a->kv_rows, a->kv_heads))
        return -1;
    for (const HeadsRef* r : {&a->q, &a->k, &a->v, &a->out})
        if ((uintptr_t)r->base % 16 || r->token % 8 || r->head % 8) return -2;
    if (!apart(a->out, a->tokens, a->heads, a->dim)) return -2;
    if (a->k.token > TOKEN_MAX || a->v.token > TOKEN_MAX) return -2;
    if ((uintptr_t)a->work % 16) return -2;
    return 0;
}

}  // namespace clear
}  // namespace pch

using namespace pch;
using namespace pch::clear;

extern "C" uint64_t pcx_attention_workspace(const AttentionArgs* a) {
    (void)a;
    return 0;
}

extern "C" int pcx_attention(const AttentionArgs* a, pc_stream_t s) {
    if (int e = checked(a)) return e;
    if (!a->tokens || !a->seqs || !a->heads) return 0;
    if (a->type == PCX_BF16)
        hipLaunchKernelGGL(attend_k<bf16>, dim3(a->tokens, a->heads), dim3(BX), 0, (hipStream_t)s, *a);
    else
        hipLaunchKernelGGL(attend_k<f16>, dim3(a->tokens, a->heads), dim3(BX), 0, (hipStream_t)s, *a);
    return launch_rc();
}
