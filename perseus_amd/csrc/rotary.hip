// Rotary positions, and the norms of queries and keys with the rotation in the same pass (pcx_rotary,
// pcx_qk_norm_rotary).
//
// Per head x of dim values: n = x w / sqrt(mean(x^2) + eps) (the norm, where wanted), then the pairs i < rot / 2 turn,
// (a, b) -> (a c - b s, b c + a s) with (c, s) = table[position][i]. Sums, squares and products are in f32; a value is
// rounded once, when it is stored.
#include "clear.h"

namespace pch {
namespace clear {

// One pass over the heads of q, then k, then v (copied): rotary alone is q without a norm.
struct Pass {
    HeadsRef in[3], out[3];
    const float* w[2];
    const int32_t* positions;
    const float* table;
    const int64_t* slots;
    int64_t places, cache_rows;
    int32_t tokens, heads, kv_heads, total, dim, rot;
    float sign, eps;
};

constexpr int WAVES = 4;

// a wave per head, a lane per pair or copied value
template <class T, bool NORM, bool INTER>
__global__ void __launch_bounds__(64 * WAVES) heads_k(Pass A) {
    const int lane = threadIdx.x & 63;
    const int64_t items = (int64_t)A.tokens * A.total;
    for (int64_t it = (int64_t)blockIdx.x * WAVES + (threadIdx.x >> 6); it < items; it += (int64_t)gridDim.x * WAVES) {
        const int64_t t = it / A.total;
        const int hh = (int)(it - t * A.total);
        const int which = hh < A.heads ? 0 : hh < A.heads + A.kv_heads ? 1 : 2;
        const int h = hh - (which == 0 ? 0 : which == 1 ? A.heads : A.heads + A.kv_heads);
        int64_t row = t;
        if (which && A.slots) {
            row = A.slots[t];
            if (row < 0 || row >= A.cache_rows) continue;
        }
        const T* x = at<T>(A.in[which], t, h);
        T* y = at<T>(A.out[which], row, h);
        if (which == 2) {
            for (int d = lane; d < A.dim; d += 64) y[d] = x[d];
            continue;
        }
        float g = 1;
        if (NORM) {
            float sum = 0;
            for (int d = lane; d < A.dim; d += 64) sum = fmaf((float)x[d], (float)x[d], sum);
            for (int m = 32; m; m >>= 1) sum += __shfl_xor(sum, m);
            g = 1.0f / sqrtf(sum / A.dim + A.eps);
        }
        const float* w = NORM ? A.w[which] : nullptr;
        const int half = A.rot >> 1;
        const int64_t pos = half ? A.positions[t] : 0;
        const bool in = half && pos >= 0 && pos < A.places;
        for (int i = lane; i < half; i += 64) {
            const int a = INTER ? 2 * i : i, b = INTER ? 2 * i + 1 : i + half;
            const float c = in ? A.table[(pos * half + i) * 2] : __builtin_nanf("");
            const float s = in ? A.table[(pos * half + i) * 2 + 1] * A.sign : __builtin_nanf("");
            const float xa = (float)x[a] * g * (w ? w[a] : 1.0f), xb = (float)x[b] * g * (w ? w[b] : 1.0f);
            y[a] = (T)(xa * c - xb * s);
            y[b] = (T)(xb * c + xa * s);
        }
        for (int d = A.rot + lane; d < A.dim; d += 64) y[d] = (T)((float)x[d] * g * (w ? w[d] : 1.0f));
    }
}

template <class T, bool NORM>
static int run_t(const Pass& a, bool inter, hipStream_t s) {
    const int64_t items = (int64_t)a.tokens * a.total;
    const int64_t blocks = (items + WAVES - 1) / WAVES;
    const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)));
    if (inter)
        hipLaunchKernelGGL((heads_k<T, NORM, true>), grid, dim3(64 * WAVES), 0, s, a);
    else
        hipLaunchKernelGGL((heads_k<T, NORM, false>), grid, dim3(64 * WAVES), 0, s, a);
    return launch_rc();
}

static int run(const Pass& a, bool norm, bool inter, int type, pc_stream_t s) {
    if ((int64_t)a.tokens * a.total == 0) return 0;
    const hipStream_t st = (hipStream_t)s;
    switch (type) {
    case PCX_BF16: return norm ? run_t<bf16, true>(a, inter, st) : run_t<bf16, false>(a, inter, st);
    case PCX_F16: return norm ? run_t<f16, true>(a, inter, st) : run_t<f16, false>(a, inter, st);
    default: return norm ? run_t<float, true>(a, inter, st) : run_t<float, false>(a, inter, st);
    }
}

// the rotation's own arguments: 0, or the error
static int rotation(int dim, int rot, int type, int64_t places, const void* positions, const void* table, int tokens) {
    if (type < PCX_BF16 || type > PCX_F32) return -1;
    if (dim < 1 || dim > 512 || rot < 0 || rot > dim || (rot & 1)) return -2;
    if (rot && (places < 0 || (tokens && (!positions || !table)))) return -1;
    return 0;
}

}  // namespace clear
}  // namespace pch

using namespace pch::clear;

extern "C" int pcx_rotary(const RotaryArgs* a, pc_stream_t s) {
    if (!a || a->tokens < 0 || a->heads < 0) return -1;
    if (int e = rotation(a->dim, a->rot, a->type, a->places, a->positions, a->table, a->tokens)) return e;
    if (!usable(a->x, a->tokens, a->heads) || !usable(a->out, a->tokens, a->heads)) return -1;
    if (!apart(a->out, a->tokens, a->heads, a->dim)) return -2;
    Pass p = {};
    p.in[0] = a->x;
    p.out[0] = a->out;
    p.positions = a->positions;
    p.table = a->table;
    p.places = a->places;
    p.tokens = a->tokens;
    p.heads = p.total = a->heads;
    p.dim = a->dim;
    p.rot = a->rot;
    p.sign = a->inverse ? -1.0f : 1.0f;
    return run(p, false, a->interleaved, a->type, s);
}

extern "C" int pcx_qk_norm_rotary(const QkNormRotaryArgs* a, pc_stream_t s) {
    if (!a || a->tokens < 0 || a->heads < 0 || a->kv_heads < 0 || !(a->eps >= 0)) return -1;
    if (int e = rotation(a->dim, a->rot, a->type, a->places, a->positions, a->table, a->tokens)) return e;
    const bool copies = a->v.base != nullptr;
    const int64_t rows = a->slots ? a->cache_rows : a->tokens;
    if (a->slots && a->cache_rows < 0) return -1;
    if (!usable(a->q, a->tokens, a->heads) || !usable(a->q_out, a->tokens, a->heads)) return -1;
    if (!usable(a->k, a->tokens, a->kv_heads) || !usable(a->k_out, rows, a->kv_heads)) return -1;
    if (copies && (!usable(a->v, a->tokens, a->kv_heads) || !usable(a->v_out, rows, a->kv_heads))) return -1;
    if (!apart(a->q_out, a->tokens, a->heads, a->dim) || !apart(a->k_out, rows, a->kv_heads, a->dim) ||
        (copies && !apart(a->v_out, rows, a->kv_heads, a->dim)))
        return -2;
    if ((int64_t)a->heads + 2 * (int64_t)a->kv_heads > 0x7fffffff) return -2;
    Pass p = {};
    p.in[0] = a->q, p.in[1] = a->k, p.in[2] = a->v;
    p.out[0] = a->q_out, p.out[1] = a->k_out, p.out[2] = a->v_out;
    p.w[0] = a->q_weight, p.w[1] = a->k_weight;
    p.positions = a->positions;
    p.table = a->table;
    p.slots = a->slots;
    p.places = a->places;
    p.cache_rows = a->cache_rows;
    p.tokens = a->tokens;
    p.heads = a->heads;
    p.kv_heads = a->kv_heads;
    p.total = a->heads + (copies ? 2 : 1) * a->kv_heads;
    p.dim = a->dim;
    p.rot = a->rot;
    p.sign = 1;
    p.eps = a->eps;
    return run(p, true, a->interleaved, a->type, s);
}
