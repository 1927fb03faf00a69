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

// ------------------------------------------------------------------------------------------------ 16 values a lane
// Two units of 8 values (16 bytes of a 16-bit type) to a lane: the two that hold its pairs' halves, or neighbours where pairs
// are neighbours. A power of two of lanes takes a head, a wave as many heads of one token as fit: short waves, many of them (a
// wave that went on to a second and third eight of heads, or a second token, kept fewer loads on their way: 16384 tokens x 40
// heads 90 to 137 us where this took 84). The bound is the memory: 8191 tokens x 40 heads of 128 in 16 bits 35 us, 4.8 TB/s (a
// large copy: 5.6); 16384 x 8 heads in 32 bits 29 us, 4.9; with the norms, 16384 x 40 heads out of rows of 48: 78 us, 4.4, and
// all 48, keys and values to rows of a cache: 97 us, 4.25.
template <class T>
struct Eight {
    float v[8];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (sizeof(T) == 2) {
            typedef T t8 __attribute__((ext_vector_type(8)));
            const t8 x = *(const t8*)p;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = (float)x[i];
        } else {
            const float4 x = ((const float4*)p)[0], y = ((const float4*)p)[1];
            v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
        }
    }
    template <bool PAST>
    __device__ __forceinline__ void store(T* p) const {
        constexpr int PER = 16 / sizeof(T);
        typedef T tv __attribute__((ext_vector_type(PER)));
#pragma unroll
        for (int k = 0; k < 8; k += PER) {
            tv x;
#pragma unroll
            for (int i = 0; i < PER; ++i) x[i] = (T)v[k + i];
            if constexpr (PAST)
                __builtin_nontemporal_store(x, (tv*)(p + k));
            else
                *(tv*)(p + k) = x;
        }
    }
};

template <class T, bool NORM, bool INTER, bool PAST>
__global__ void __launch_bounds__(64 * WAVES) units_k(Pass A, int lph_log, uint32_t chunks) {
    const int lane = threadIdx.x & 63, lph = 1 << lph_log, slot = lane >> lph_log, l = lane & (lph - 1);
    const uint32_t wv = blockIdx.x * WAVES + (threadIdx.x >> 6), t = wv / chunks;
    const int hh = (int)(wv - t * chunks) * (64 >> lph_log) + slot;
    if (t >= (uint32_t)A.tokens || hh >= A.total) return;  // whole heads: the lanes of one leave together
    // q, k or v by selects: an indexed kernel argument would be a load, and the first load waits for it
    const bool isq = !NORM || hh < A.heads, isv = NORM && hh >= A.heads + A.kv_heads;
    const int h = isq ? hh : isv ? hh - A.heads - A.kv_heads : hh - A.heads;
    const HeadsRef in = isq ? A.in[0] : isv ? A.in[2] : A.in[1], out = isq ? A.out[0] : isv ? A.out[2] : A.out[1];
    const int units = A.dim >> 3, turned = isv ? 0 : A.rot >> 3;
    // this lane's units, and whether they turn
    int ua, ub;
    bool ta, tb;
    if (INTER) {
        ua = 2 * l, ub = 2 * l + 1;
        ta = ua < turned, tb = ub < turned;
    } else {
        const int half = turned >> 1;
        ta = tb = l < half;
        ua = ta ? l : turned + 2 * (l - half);
        ub = ta ? l + half : ua + 1;
    }
    const bool va = ua < units, vb = ub < units;
    Eight<T> a, b;
#pragma unroll
    for (int i = 0; i < 8; ++i) a.v[i] = b.v[i] = 0;
    const T* x = at<T>(in, t, h);
    if (va) a.load(x + 8 * ua);
    if (vb) b.load(x + 8 * ub);
    int64_t row = t;
    if (NORM && !isq && A.slots) {
        row = A.slots[t];
        if (row >= A.cache_rows) row = -1;
    }
    float c[8], s[8];  // of this lane's pairs
    if (ta) {
        const int64_t pos = A.positions[t];
        const bool inside = pos >= 0 && pos < A.places;
        const float4* tab = (const float4*)(A.table + (inside ? pos : 0) * A.rot) + (INTER ? ua * 2 : l * 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float nan = __builtin_nanf("");
            const float4 y = !inside ? make_float4(nan, nan, nan, nan) : !INTER || i < 2 || tb ? tab[i] : make_float4(1, 0, 1, 0);
            c[2 * i] = y.x, c[2 * i + 1] = y.z;
            s[2 * i] = y.y * A.sign, s[2 * i + 1] = y.w * A.sign;
        }
    }
    if (NORM && !isv) {
        const float* w = isq ? A.w[0] : A.w[1];
        Eight<float> wa, wb;
#pragma unroll
        for (int i = 0; i < 8; ++i) wa.v[i] = wb.v[i] = 1;
        if (w && va) wa.load(w + 8 * ua);
        if (w && vb) wb.load(w + 8 * ub);
        float sum = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fmaf(a.v[i], a.v[i], fmaf(b.v[i], b.v[i], sum));
        for (int m = 1; m < lph; m <<= 1) sum += __shfl_xor(sum, m);
        const float g = 1.0f / sqrtf(sum / A.dim + A.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) a.v[i] *= g * wa.v[i], b.v[i] *= g * wb.v[i];
    }
    if (row < 0) return;
    if (ta)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float& x0 = INTER ? (i < 4 ? a.v[2 * i] : b.v[2 * i - 8]) : a.v[i];
            float& x1 = INTER ? (i < 4 ? a.v[2 * i + 1] : b.v[2 * i - 7]) : b.v[i];
            const float y0 = x0 * c[i] - x1 * s[i], y1 = x1 * c[i] + x0 * s[i];
            if (!INTER || i < 4 || tb) x0 = y0, x1 = y1;
        }
    T* y = at<T>(out, row, h);
    if (va) a.template store<PAST>(y + 8 * ua);
    if (vb) b.template store<PAST>(y + 8 * ub);
}

// ------------------------------------------------------------------------------------------------ any size
// Odd sizes, strides and addresses, what 16-byte accesses do not fit: a wave per head, a lane per pair or copied value. Halves
// that are not whole units of 8 too (rot 8, 24, 40, 72 in the half layout): 8191 tokens x 40 heads of 128, rot 24, 114 us (150
// with three inputs in turn) where units_k takes 36 with rot 32.
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

// whether units_k's 16-byte accesses and whole units fit
template <class T>
static bool whole_units(const Pass& a, bool inter) {
    constexpr int per = 16 / (int)sizeof(T);
    if (a.dim % 8 || a.rot % (inter ? 8 : 16)) return false;
    if (((uintptr_t)a.table | (uintptr_t)a.w[0] | (uintptr_t)a.w[1]) % 16) return false;
    for (int i = 0; i < 3; ++i)
        for (const HeadsRef* r : {&a.in[i], &a.out[i]})
            if (r->base && ((uintptr_t)r->base % 16 || r->token % per || r->head % per)) return false;
    return true;
}

template <class T, bool NORM, bool INTER>
static int run_t(const Pass& a, hipStream_t s) {
    if (whole_units<T>(a, INTER)) {
        int lph_log = 0;
        while (16 << lph_log < a.dim) ++lph_log;
        const int slots = 64 >> lph_log, all = (a.total + slots - 1) / slots;
        const int64_t blocks = ((int64_t)a.tokens * all + WAVES - 1) / WAVES;
        // outputs that no L2 holds until they are read go past the caches: 84 MB 38.5 -> 35.3 us, 168 MB 83 -> 78
        const bool past = (int64_t)a.tokens * a.total * a.dim * sizeof(T) > 32 << 20;
        if (blocks < 1 << 24) {  // fewer than 2^32 threads: more no launch takes, and heads_k goes on by itself
            const dim3 grid((unsigned)blocks);
            if (past)
                hipLaunchKernelGGL((units_k<T, NORM, INTER, true>), grid, dim3(64 * WAVES), 0, s, a, lph_log, (uint32_t)all);
            else
                hipLaunchKernelGGL((units_k<T, NORM, INTER, false>), grid, dim3(64 * WAVES), 0, s, a, lph_log, (uint32_t)all);
            return launch_rc();
        }
    }
    const int64_t items = (int64_t)a.tokens * a.total;
    const int64_t blocks = (items + WAVES - 1) / WAVES;
    const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)));
    hipLaunchKernelGGL((heads_k<T, NORM, INTER>), grid, dim3(64 * WAVES), 0, s, a);
    return launch_rc();
}

template <class T>
static int run_l(const Pass& a, bool norm, bool inter, hipStream_t s) {
    if (norm) return inter ? run_t<T, true, true>(a, s) : run_t<T, true, false>(a, s);
    return inter ? run_t<T, false, true>(a, s) : run_t<T, false, false>(a, s);
}

static int run(const Pass& a, bool norm, bool inter, int type, pc_stream_t s) {
    if ((int64_t)a.tokens * a.total == 0) return 0;
    const hipStream_t st = (hipStream_t)s;
    switch (type) {
    case PCX_BF16: return run_l<bf16>(a, norm, inter, st);
    case PCX_F16: return run_l<f16>(a, norm, inter, st);
    default: return run_l<float>(a, norm, inter, st);
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
    p.in[0] = settled(a->x, a->tokens, a->heads, a->dim);
    p.out[0] = settled(a->out, a->tokens, a->heads, a->dim);
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
    p.in[0] = settled(a->q, a->tokens, a->heads, a->dim), p.out[0] = settled(a->q_out, a->tokens, a->heads, a->dim);
    p.in[1] = settled(a->k, a->tokens, a->kv_heads, a->dim), p.out[1] = settled(a->k_out, rows, a->kv_heads, a->dim);
    p.in[2] = settled(a->v, a->tokens, a->kv_heads, a->dim), p.out[2] = settled(a->v_out, rows, a->kv_heads, a->dim);
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
