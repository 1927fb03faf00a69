// Attention of packed sequences over keys and values that lie packed or in caches (pcx_attention).
//
// For a query q that sees the keys j: z_j = scale q . k_j, m = max z_j, l = sum exp(z_j - m), o = sum exp(z_j - m) v_j / l,
// lse = m + log l. One pass over the keys holds (m, l, o) and rescales l and o where m grows. Scores, exponentials, sums and o are
// f32; the weights exp(z_j - m) are rounded to the type for their product with v, which the matrix cores take, and l sums them
// unrounded. That rounding costs about as much again as the output's own (2^-8 of a weight at most for bf16, 2^-11 for f16: the
// error against 64 bits is 1.1 to 1.4 times that of one rounding). Where few_k takes rows of a token or a few, which are bound by
// the reading of the keys, what it leaves is a second product, and the error is that of the output's rounding alone; a second
// product in rows_k, which is bound by its products, would be half as many again.
//
// few_k takes the rows of tokens, up to 128 of a key head where they are few tiles, and the prompts of 64 dimensions whose tiles
// of 128 rows would not fill the chip, and splits the keys over waves and workgroups; rows_k takes all others (prompts, chunks) in
// tiles of 128 rows; join_k joins the parts of both. The rules and their measurements stand at choose().
//
// The rows of a tile are the (query, head) pairs of one key head, numbered query * group + head of the group: a tile of rows
// reads its keys once for the whole group, and one token of a wide group fills a tile as a run of queries does. Everything is
// transposed so that a lane holds one row: the 32 x 32 products z^T = K q^T leave in lane (c, h) (c = lane mod 32, h =
// lane / 32) the scores of row c with the keys 8 i + 4 h + j (i, j < 4), so that row statistics are sums inside a lane and
// one exchange between the two halves, and the probabilities are already the right operand of o^T += V^T p^T if V's keys
// are taken in that order: the transposing LDS read gives four keys of a column to a lane, which is that order.
#include <algorithm>

#include "clear.h"

namespace pch {
namespace clear {

constexpr int DMAX = 256;
constexpr int64_t TOKEN_MAX = 1 << 22;  // key rows' distance, in elements: a tile's byte offsets stay in 32 bits
constexpr int64_t ROWS_MAX = 0x7fffffff - 127;  // query heads: the last row of a tile of 128 stays in 31 bits
constexpr int64_t ITEMS_MAX = 0x7fffffff - 65535;  // (sequence, tile, part): their number in a grid of rows of 65535
constexpr int32_t KV_HEADS_MAX = (1 << 23) - 1;  // a grid's threads in one dimension, 512 to a key head: below 2^32

typedef float v16f __attribute__((ext_vector_type(16)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef float v8f __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
#define PCH_LDS __attribute__((address_space(3)))

// BELOW: how far under a row's largest score (log2 units) the m is kept that its weights exp2(z - m) are taken from. f16 ends
// at 2^-25, half its smallest step: with m at the largest score 31 weights of 2^-25.2 beside a 1 were lost whole (an output of
// 8.7e-4 came as 0); 7 below they begin at 2^-32 of the largest, and end, m lagging by up to 8, at 2^15, within f16.
template <class T>
struct Mat;
template <>
struct Mat<bf16> {
    typedef bf16 v8 __attribute__((ext_vector_type(8)));
    typedef bf16 v4 __attribute__((ext_vector_type(4)));
    static constexpr float BELOW = 0;
    static __device__ __forceinline__ v16f mul(v8 a, v8 b, v16f c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Mat<f16> {
    typedef f16 v8 __attribute__((ext_vector_type(8)));
    typedef f16 v4 __attribute__((ext_vector_type(4)));
    static constexpr float BELOW = 7;
    static __device__ __forceinline__ v16f mul(v8 a, v8 b, v16f c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};

// the other half's value of a lane's row
__device__ __forceinline__ float other(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    // r[0]: the low half's value in both halves, r[1]: the high half's
    return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

// ------------------------------------------------------------------------------------------------ tiles of keys
// KT rows of room for DP values in LDS (of which the products take DC), 16-byte chunks permuted within a row so that both
// readings are free of bank conflicts: keys (16 lanes take one chunk of 16 rows) by xor with the row number, values (32 lanes of
// the transposing read take 64 bytes of 4 rows) by xor with four times the row number (twice it: 67 million conflict cycles at
// 16384 tokens x 16 heads; so: none).
template <int DP>
struct Tile {
    static constexpr int CPR = DP / 8;  // chunks of a row
    static __device__ __forceinline__ int kswz(int key) { return DP == 64 ? (key >> 1) & 7 : key & 15; }
    static __device__ __forceinline__ int vswz(int key) { return DP == 64 ? 4 * ((key >> 1) & 1) : 4 * (key & 3); }
};

// 64 lanes' 16 bytes each from a buffer into LDS at `lds` + 16 lane, N times, STEP bytes of LDS apart; lanes past the buffer's
// end write zeros. It counts in vmcnt like a load; nothing waits for it but the caller's own s_waitcnt (the builtin's loads are
// waited for, all of them, before the next LDS reading, the tiles on their way too). The operands' scalar registers may have
// been written by vector instructions (a spilled one is read back by v_readlane): five states until a buffer instruction may
// read them, and one after m0.
template <int STEP, int N>
__device__ __forceinline__ void load_lds(__amdgpu_buffer_rsrc_t r, uint32_t lds, const uint32_t (&off)[N]) {
    static_assert(N == 2 || N % 4 == 0);
    if constexpr (N == 2) {
        asm volatile(
            "s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %3, 0 offen lds\n\t"
            "s_add_u32 m0, m0, %4\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds"
            :
            : "s"(lds), "v"(off[0]), "v"(off[1]), "s"(r), "n"(STEP)
            : "memory", "m0", "scc");
    } else {
#pragma unroll
        for (int n = 0; n < N; n += 4)
            asm volatile(
                "s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %5, 0 offen lds\n\t"
                "s_add_u32 m0, m0, %6\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %5, 0 offen lds\n\t"
                "s_add_u32 m0, m0, %6\n\ts_nop 0\n\tbuffer_load_dwordx4 %3, %5, 0 offen lds\n\t"
                "s_add_u32 m0, m0, %6\n\ts_nop 0\n\tbuffer_load_dwordx4 %4, %5, 0 offen lds"
                :
                : "s"(lds + n * STEP), "v"(off[n]), "v"(off[n + 1]), "v"(off[n + 2]), "v"(off[n + 3]), "s"(r), "n"(STEP)
                : "memory", "m0", "scc");
    }
}

// All loads are there, the compiler's own among them. It counts those alone: one of its loads before a loop (a query's, the rare
// repair's) that it does not know to be there makes it wait for everything, the tiles on their way too, in every step.
__device__ __forceinline__ void settled() { __builtin_amdgcn_s_waitcnt(0x0f70); }

// log of a row's sum l of exp2(. - m), in natural units; no key: l = 0 gives -infinity
__device__ __forceinline__ float logsum(float m, float l) {
    return l == 0.0f ? -INFINITY : (m + __log2f(l)) * 0.6931471805599453f;
}

__device__ __forceinline__ uint64_t uniform64(uint64_t v) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return ((uint64_t)hi << 32) | lo;
}

// rows of one (sequence, key head): what a workgroup works on
struct Work {
    int q0, n;       // query rows of the sequence
    int64_t k0;      // its first key row
    int len;         // its keys
    int tile;        // tile of rows
    int chunk, nc;   // part of the tile's keys, and how many parts they are split into
    int slot;        // where the tile's partial sums begin
    bool live;
};

// How a launch splits keys: a sequence of len keys into ceil(len / size) parts, most at the most. Lengths beyond what the
// caller expected only make the parts longer.
struct Split {
    int most, size;
    int* arrived;  // [tile][kv head] parts that are done, zero between calls; null: join_k joins them
    float* work;   // [slot][BM][dim] sums, then [slot][BM][2] maxima and weights' sums
    int64_t slots;
    __device__ __forceinline__ int parts(int len) const {
        if (most <= 1) return 1;
        const int n = (int)(((uint32_t)len + size - 1) / (uint32_t)size);
        return n < 1 ? 1 : n < most ? n : most;
    }
    __device__ __forceinline__ float* sums(int slot, int BM, int dim) const { return work + (int64_t)slot * BM * dim; }
    __device__ __forceinline__ float* stats(int slot, int BM, int dim) const {
        return work + slots * BM * dim + (int64_t)slot * BM * 2;
    }
};

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

// tiles of KT keys that n keys take, and the keys of so many tiles: up to 2^31, one more than an int holds
template <int KT>
__device__ __forceinline__ int tiles_of(int n) {
    return (int)(((uint32_t)n + KT - 1) / KT);
}
template <int KT>
__device__ __forceinline__ int keys_of(int tiles, int most) {
    return (int)min((uint32_t)tiles * KT, (uint32_t)most);
}

// inclusive sums over the lanes of a wave, and the largest value (by data-parallel moves: no trip through LDS)
template <int CTRL, int ROWS>
__device__ __forceinline__ int moved(int x) {
    return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int lane_sums(int x) {
    x += moved<0x111, 0xf>(x);  // from 1, 2, 4 and 8 lanes below in a row of 16
    x += moved<0x112, 0xf>(x);
    x += moved<0x114, 0xf>(x);
    x += moved<0x118, 0xf>(x);
    x += moved<0x142, 0xa>(x);  // the last lane of rows 0 and 2 into rows 1 and 3
    x += moved<0x143, 0xc>(x);  // lane 31 into rows 2 and 3
    return x;
}
__device__ __forceinline__ int total(int x) { return __builtin_amdgcn_readlane(lane_sums(x), 63); }
__device__ __forceinline__ int largest(int x) {  // of values not negative
    x = max(x, moved<0x111, 0xf>(x));
    x = max(x, moved<0x112, 0xf>(x));
    x = max(x, moved<0x114, 0xf>(x));
    x = max(x, moved<0x118, 0xf>(x));
    x = max(x, moved<0x142, 0xa>(x));
    x = max(x, moved<0x143, 0xc>(x));
    return __builtin_amdgcn_readlane(x, 63);
}

// item -> (sequence, tile of BM rows, part of its keys); BYPART false: all parts of a tile in one item. Every wave finds it by
// itself, a lane per sequence. BYLEVEL: the tiles of up to 64 sequences go longest first (a tile's level: its keys in units of
// its rows' queries), as workgroups start in their order and a long one that starts last is waited for (48 caches of 89 to 8000
// keys, one token each: 174 -> 159 us); else, and for more sequences, one sequence after the other, each sequence's last tile
// first.
template <bool BYPART, bool BYLEVEL>
__device__ __forceinline__ Work locate(const AttentionArgs& A, const Split& S, int item, int group, int BM) {
    const int lane = threadIdx.x & 63;
    Work w;
    w.live = false;
    for (int base = 0; base < A.seqs; base += 64) {
        const int b = base + lane;
        int q0 = 0, n = 0, len = 0;
        int64_t k0 = 0;
        if (b < A.seqs) {
            q0 = clampi(A.q_start[b], 0, A.tokens);
            n = clampi(A.q_start[b + 1], 0, A.tokens) - q0;
            n = n < 0 ? 0 : n;
            k0 = A.k_start[b];
            len = A.k_len[b];
            if (k0 < 0 || k0 >= A.kv_rows) k0 = len = 0;
            if (len < 0) len = 0;
            if (len > A.kv_rows - k0) len = (int)(A.kv_rows - k0);
        }
        const int parts = S.parts(len), tiles = (int)(((int64_t)n * group + BM - 1) / BM), nc = BYPART ? parts : 1;
        int src = 0, at;  // the lane of the item's sequence, and its number there
        if (A.seqs == 1) {
            const int all = __builtin_amdgcn_readfirstlane(tiles * nc);
            if (item >= all) return w;
            w.nc = __builtin_amdgcn_readfirstlane(parts);
            at = all - 1 - item;
            w.tile = BYPART && w.nc > 1 ? at / w.nc : at;
            w.chunk = BYPART ? at - w.tile * w.nc : 0;
        } else if (BYLEVEL && A.seqs <= 64) {
            // a tile's level is `above` + its number, or (not causal) `above`
            const int keys = A.causal ? (len > n ? len - n : 0) : len;
            // (a bound that only matters to the order: no sum of levels leaves 31 bits)
            const int above = (int)std::min<int64_t>((int64_t)keys * group / BM, 1 << 30), span = A.causal ? tiles : tiles > 0;
            const int each = A.causal ? nc : tiles * nc;
            // the items of a lane's own level u and more
            const auto count = [&](int u) {
                int c = 0;
                for (int x = 0; x < A.seqs; ++x) {
                    const int sp = __builtin_amdgcn_readlane(span, x), to = __builtin_amdgcn_readlane(above, x) + sp;
                    c += clampi(to - u, 0, sp) * __builtin_amdgcn_readlane(each, x);
                }
                return c;
            };
            // the largest level that has more than `item` items from it on: 64 levels at a time
            int lo = 0, step = largest(above + span), over = 0;
            do {
                step = (step + 63) >> 6;
                const int c = count(lo + lane * step);
                const uint64_t past = __ballot(c > item);
                if (!past) return w;
                const int l = 63 - __builtin_clzll(past);
                over = l < 63 ? __builtin_amdgcn_readlane(c, l + 1) : -1;
                lo += l * step;
            } while (step > 1);
            if (over < 0) over = __builtin_amdgcn_readfirstlane(count(lo + 1));
            item -= over;
            const int own = (clampi(above + span - lo, 0, span) - clampi(above + span - lo - 1, 0, span)) * each;
            const int sum = lane_sums(lane < A.seqs ? own : 0);
            src = __builtin_ctzll(__ballot(sum > item));
            at = item - __builtin_amdgcn_readlane(sum - own, src);
            w.nc = __builtin_amdgcn_readlane(parts, src);
            w.tile = A.causal ? lo - __builtin_amdgcn_readlane(above, src) : BYPART && w.nc > 1 ? at / w.nc : at;
            w.chunk = !BYPART ? 0 : A.causal ? at : at - w.tile * w.nc;
        } else {
            const int sum = lane_sums(tiles * nc);
            const uint64_t past = __ballot(sum > item);
            if (!past) {
                item -= __builtin_amdgcn_readlane(sum, 63);
                continue;
            }
            src = __builtin_ctzll(past);
            w.nc = __builtin_amdgcn_readlane(parts, src);
            at = __builtin_amdgcn_readlane(sum, src) - 1 - item;
            w.tile = BYPART && w.nc > 1 ? at / w.nc : at;
            w.chunk = BYPART ? at - w.tile * w.nc : 0;
        }
        w.q0 = __builtin_amdgcn_readlane(q0, src);
        w.n = __builtin_amdgcn_readlane(n, src);
        w.len = __builtin_amdgcn_readlane(len, src);
        const uint32_t k_lo = __builtin_amdgcn_readlane((int)(uint32_t)k0, src);
        const uint32_t k_hi = __builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)k0 >> 32), src);
        w.k0 = (int64_t)(((uint64_t)k_hi << 32) | k_lo);
        // tiles of different sequences apart: a sequence has at most one tile more than its rows divided by BM
        w.slot = S.most > 1 ? ((int)((int64_t)w.q0 * group / BM) + base + src + w.tile) * S.most : 0;
        w.live = true;
        return w;
    }
    return w;
}

// rows are numbered query * group + head of the group; exact for every int
struct Group {
    int n;
    double inv;
    __device__ __forceinline__ int query(int row) const { return (int)(((double)row + 0.5) * inv); }
};

// the keys that row r of the sequence sees (the last row's where r is past it, so that unused rows need no masks)
__device__ __forceinline__ int seen(const Work& w, int r, const Group& group, int causal) {
    if (!causal) return w.len;
    int i = __builtin_amdgcn_readfirstlane(group.query(r));
    i = i < w.n ? i : w.n - 1;
    return clampi(w.len - w.n + i + 1, 0, w.len);
}

// ------------------------------------------------------------------------------------------------ a wave's rows
// 32 rows of a wave: queries, running statistics and o^T (lane (c, h): row c, dimensions 32 db + 8 i + 4 h + j)
template <class T, int DC>
struct Rows {
    typename Mat<T>::v8 q[DC / 16];
    v16f o[DC / 32];
    float m, nm, l;  // running maximum less BELOW (log2 units), its negative (0 where there is none yet), this half's sum
    int lim;         // keys seen

    // row: this lane's in the sequence (past the last one: the last one's again, its result not kept)
    __device__ __forceinline__ void begin(const AttentionArgs& A, const Work& w, int kvh, const Group& group, int row) {
        const int h = (threadIdx.x & 63) >> 5;
        int i = group.query(row), hd = kvh * group.n + (row - i * group.n);
        if (i >= w.n) i = w.n - 1, hd = kvh * group.n;
        const T* x = at<T>(A.q, w.q0 + i, hd);
#pragma unroll
        for (int s = 0; s < DC / 16; ++s) {
            const int d = 16 * s + 8 * h;
            if (16 * s + 16 <= A.dim)
                q[s] = *(const typename Mat<T>::v8*)(x + d);
            else
                q[s] = d < A.dim ? *(const typename Mat<T>::v8*)(x + d) : (typename Mat<T>::v8)(T)0.0f;
        }
#pragma unroll
        for (int d = 0; d < DC / 32; ++d) o[d] = (v16f)0.0f;
        m = -INFINITY;
        nm = 0;
        l = 0;
        lim = A.causal ? clampi(w.len - w.n + i + 1, 0, w.len) : w.len;
    }
};

template <class T, int DP, int DC, int KT>
struct Wave {
    typedef typename Mat<T>::v8 v8;
    static constexpr int NK = KT / 32;
    using L = Tile<DP>;

    // scores of KT keys: z[kb] for the keys 32 kb ..
    template <bool ALONE = true>
    static __device__ __forceinline__ void scores(const char PCH_LDS* k, const Rows<T, DC>& R, v16f (&z)[NK]) {
        const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
        const uint32_t row = c * DP * 2;
#pragma unroll
        for (int kb = 0; kb < NK; ++kb) z[kb] = (v16f)0.0f;
#pragma unroll
        for (int s = 0; s < DC / 16; ++s) {
#pragma unroll
            for (int kb = 0; kb < NK; ++kb) {
                const v8 a = *(const v8 PCH_LDS*)(k + row + kb * 32 * DP * 2 + (((2 * s + h) ^ L::kswz(c)) << 4));
                z[kb] = Mat<T>::mul(a, R.q[s], z[kb]);
            }
        }
        // four readings ahead of the products
        if (!ALONE) return;
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
        for (int x = 0; x < NK * DC / 16 - 4; ++x) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x8, 4, 0);
    }

    // keys from the row's limit on do not count; key0: the tile's first
    static __device__ __forceinline__ void mask(const Rows<T, DC>& R, int key0, v16f (&z)[NK]) {
        const int left = R.lim - key0 - 4 * ((threadIdx.x & 63) >> 5);
#pragma unroll
        for (int kb = 0; kb < NK; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                if (32 * kb + 8 * (e >> 2) + (e & 3) >= left) z[kb][e] = -INFINITY;
                if ((e & 3) == 3) __builtin_amdgcn_sched_barrier(0);  // not all comparisons at once: they would not fit
            }
    }

    // z becomes exp2(c z - m); m follows the largest score where it has grown by more than 8 (2^8 times as much holds in every
    // type, and most tiles then need no rescaling)
    static __device__ __forceinline__ void softmax(Rows<T, DC>& R, float c, v16f (&z)[NK]) {
        grow(R, c, largest_of(z));
        weigh(R, c, z);
    }
    static __device__ __forceinline__ float largest_of(const v16f (&z)[NK]) {
        float top = z[0][0];
#pragma unroll
        for (int kb = 0; kb < NK; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e) top = fmaxf(top, z[kb][e]);
        return top;
    }
    static __device__ __forceinline__ void grow(Rows<T, DC>& R, float c, float top) {
        top = fmaf(fmaxf(top, other(top)), c, -Mat<T>::BELOW);
        if (__any(top > R.m + 8.0f)) {
            const float mn = fmaxf(R.m, top);
            const float r = mn == R.m ? 1.0f : __builtin_amdgcn_exp2f(R.m - mn);
            R.m = mn;
            R.nm = mn == -INFINITY ? 0.0f : -mn;
            R.l *= r;
#pragma unroll
            for (int d = 0; d < DC / 32; ++d) R.o[d] *= r;
        }
    }
    static __device__ __forceinline__ void weigh(Rows<T, DC>& R, float c, v16f (&z)[NK]) {
        float l = 0;
#pragma unroll
        for (int kb = 0; kb < NK; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                z[kb][e] = __builtin_amdgcn_exp2f(fmaf(z[kb][e], c, R.nm));
                l += z[kb][e];
            }
        R.l += l;
    }

    // o += p V; TWICE: with what the weights' rounding left as a second product
    template <bool TWICE = false>
    static __device__ __forceinline__ void values(const char PCH_LDS* v, Rows<T, DC>& R, const v16f (&z)[NK]) {
        const int lane = threadIdx.x & 63;
        const int key = 4 * (lane >> 5) + ((lane & 15) >> 2), ch = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
        const uint32_t at = key * DP * 2 + (lane & 1) * 8;
#pragma unroll
        for (int s = 0; s < KT / 16; ++s) {
            v8f pf;
#pragma unroll
            for (int e = 0; e < 8; ++e) pf[e] = z[s >> 1][8 * (s & 1) + e];
            const v8 p = __builtin_convertvector(pf, v8);
            v8 rest;
            if (TWICE) rest = __builtin_convertvector(pf - __builtin_convertvector(p, v8f), v8);
#pragma unroll
            for (int d = 0; d < DC / 32; ++d) {
                // the swizzle of rows 8 apart is the same
                const uint32_t x = at + (((4 * d + ch) ^ L::vswz(key)) << 4) + 16 * s * DP * 2;
                const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((v4s PCH_LDS*)(v + x));
                const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((v4s PCH_LDS*)(v + x + 8 * DP * 2));
                const v8s a = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                R.o[d] = Mat<T>::mul(__builtin_bit_cast(v8, a), p, R.o[d]);
                if (TWICE) R.o[d] = Mat<T>::mul(__builtin_bit_cast(v8, a), rest, R.o[d]);
            }
        }
    }

    // The rare repair of the tiles that a row sees in part. There o^T += V^T p^T multiplies values that a row does not see by
    // zero, which is not zero where they are infinite or NaN: those of keys that later rows see, or, where rows of values share
    // memory, seen ones read again past the last key (else zeros are read there). If o came out so, o of these keys (from key0 to
    // each row's limit, a tile of KT in every `step`) is summed again from memory, key by key, each row its own.
    static __device__ __forceinline__ void repair(const AttentionArgs& A, const Work& w, int kvh, float c, uint32_t key0,
                                               uint32_t key1, uint32_t step, Rows<T, DC>& R) {
        const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
        for (int d = 0; d < DC / 32; ++d) R.o[d] = (v16f)0.0f;
        for (uint32_t t0 = key0; t0 < key1; t0 += step)
            for (uint32_t j = t0; j < t0 + KT && j < key1; ++j) {
                const T* k = at<T>(A.k, w.k0 + j, kvh);
                const T* v = at<T>(A.v, w.k0 + j, kvh);
                float z = 0;
#pragma unroll
                for (int s = 0; s < DC / 16; ++s) {
                    if (16 * s + 8 * h < A.dim) {
                        const v8 x = *(const v8*)(k + 16 * s + 8 * h);
#pragma unroll
                        for (int e = 0; e < 8; ++e) z = fmaf((float)x[e], (float)R.q[s][e], z);
                    }
                }
                z += other(z);
                if ((int)j >= R.lim) continue;
                const float p = __builtin_amdgcn_exp2f(fmaf(z, c, R.nm));
#pragma unroll
                for (int d = 0; d < DC / 32; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int dd = 32 * d + 8 * i + 4 * h;
                        if (dd < A.dim) {
                            const typename Mat<T>::v4 x = *(const typename Mat<T>::v4*)(v + dd);
#pragma unroll
                            for (int e = 0; e < 4; ++e) R.o[d][4 * i + e] = fmaf(p, (float)x[e], R.o[d][4 * i + e]);
                        }
                    }
            }
    }
    static __device__ __forceinline__ bool broken(const Rows<T, DC>& R) {
        float x[4] = {0, 0, 0, 0};
#pragma unroll
        for (int d = 0; d < DC / 32; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e & 3] = fmaf(R.o[d][e], 0.0f, x[e & 3]);
        return __any(!((x[0] + x[1]) + (x[2] + x[3]) == 0.0f));
    }

    // o / l and lse, or (a part of the keys) o, m and l; BM: rows of the tile, row: this lane's in it
    static __device__ __forceinline__ void finish(const AttentionArgs& A, const Split& S, const Work& w, int kvh,
                                                  const Group& group, int BM, int row, Rows<T, DC>& R) {
        const int h = (threadIdx.x & 63) >> 5, r = w.tile * BM + row;
        const int i = group.query(r), hd = kvh * group.n + (r - i * group.n);
        const float l = R.l + other(R.l);
        if (w.nc > 1) {
            if (i >= w.n) return;
            const int slot = (w.slot + w.chunk) * A.kv_heads + kvh;
            float* y = S.sums(slot, BM, A.dim) + (int64_t)row * A.dim;
#pragma unroll
            for (int d = 0; d < DC / 32; ++d)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int dd = 32 * d + 8 * g + 4 * h;
                    if (dd < A.dim)
                        *(v4f*)(y + dd) = v4f{R.o[d][4 * g], R.o[d][4 * g + 1], R.o[d][4 * g + 2], R.o[d][4 * g + 3]};
                }
            if (h == 0) *(float2*)(S.stats(slot, BM, A.dim) + row * 2) = make_float2(R.m, l);
            return;
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        T* y = at<T>(A.out, w.q0 + i, hd);
        typedef uint32_t v2u __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int d = 0; d < DC / 32; ++d)
#pragma unroll
            for (int g = 0; g < 4; g += 2) {
                v2u x[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int a = 4 * (g + e);
                    const v4f f = v4f{R.o[d][a], R.o[d][a + 1], R.o[d][a + 2], R.o[d][a + 3]} * inv;
                    x[e] = __builtin_bit_cast(v2u, __builtin_convertvector(f, typename Mat<T>::v4));
                }
                // the halves of a row hold 4 values each of both groups of 8: after the exchange a lane holds one group
                const auto a = __builtin_amdgcn_permlane32_swap(x[0][0], x[1][0], false, false);
                const auto b = __builtin_amdgcn_permlane32_swap(x[0][1], x[1][1], false, false);
                const int dd = 32 * d + 8 * (g + h);
                if (i < w.n && dd < A.dim) *(v4u*)(y + dd) = v4u{a[0], b[0], a[1], b[1]};
            }
        if (A.lse && h == 0 && i < w.n)
            A.lse[(int64_t)(w.q0 + i) * A.heads + hd] = logsum(R.m, l);
    }
};

// ------------------------------------------------------------------------------------------------ many rows
// A workgroup of NW waves takes 32 NW rows; a tile of keys and values goes through LDS once for all of them, the next one loaded
// while this one is used (two buffers of each: 64 KB at 128 dimensions, so that two workgroups share a CU). Tiles run from the
// last to the first: those that rows see in part come first, and if they hold infinities or NaN that some row does not see their
// sums are made again (repair) before the rest is added. The scores of tile t - 1 are made in tile t's step, beside its
// exponentials, so that a wave has matrix and vector work at once.
//
// 16384 tokens x 16 heads of 128, causal, f16: 1.02 to 1.13 ms by the card, 1080 to 970 TFLOP/s (a 16384^3 product: 1303); the
// matrix cores are busy 59% of the cycles at the 1.6 to 1.75 GHz to which the card's power takes the clock, and without any
// softmax the same products take 0.95 ms. 32 rows a wave: 64 would halve the LDS readings (256 bytes a cycle: half used) but
// spill. One wave of two a SIMD needs 2500 cycles for a step whose products take 1050 and whose vector instructions take 1100:
// two hide each other's waits (four buffers for one wave a SIMD: 197 -> 286 us, the packed prompts below). Tiles of 64 keys, 32
// above 128 dimensions, where o takes half the registers (64 at 256: 321 -> 402 us; 32 at 128: 1107 -> 1132); two waves a SIMD up
// to 192 dimensions (one: 274 us, two: 216, 2 x 4000 tokens x 16 heads), one above (two spill). Nine prompts of 269 to 2048
// tokens x 32 heads, bf16: 189 to 206 us, 850 to 780 TFLOP/s; a fifth of a workgroup's cycles is its start and end (finding its
// tile, first loads, queries, output).
template <class T, int DP, int DC, int NW>
__global__ void __launch_bounds__(64 * NW, DC > 192 ? 1 : 2) rows_k(AttentionArgs A, Split S, Group group) {
    constexpr int KT = DP > 128 ? 32 : 64, BM = 32 * NW, TB = KT * DP * 2, CPR = DP / 8, NK = KT / 32;
    constexpr int NL = KT * CPR / (64 * NW);  // loads a wave issues for a tile of keys, or of values
    using W = Wave<T, DP, DC, KT>;
    __shared__ __attribute__((aligned(1024))) char lds[4 * TB];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int kvh = blockIdx.x;
    const Work w = locate<true, true>(A, S, blockIdx.z * gridDim.y + blockIdx.y, group.n, BM);
    if (!w.live) return;
    const int R = w.n * group.n, r0 = w.tile * BM, mine = r0 + wave * 32;
    const float c = A.scale * 1.4426950408889634f;
    const int last = r0 + BM < R ? r0 + BM : R;
    const int all = tiles_of<KT>(seen(w, last - 1, group, A.causal));
    int first = 0, tiles = all;
    if (w.nc > 1) {
        first = (int)((int64_t)all * w.chunk / w.nc);
        tiles = (int)((int64_t)all * (w.chunk + 1) / w.nc);
    }

    uint32_t ko[NL], vo[NL];
#pragma unroll
    for (int n = 0; n < NL; ++n) {
        const int p = (n * NW + wave) * 64 + lane, key = p / CPR, cp = p % CPR;
        const int ck = cp ^ Tile<DP>::kswz(key), cv = cp ^ Tile<DP>::vswz(key);
        ko[n] = ck * 8 < A.dim ? key * (uint32_t)A.k.token * 2 + ck * 16 : 0x7ffffff0u;
        vo[n] = cv * 8 < A.dim ? key * (uint32_t)A.v.token * 2 + cv * 16 : 0x7ffffff0u;
    }
    const uint32_t base = (uint32_t)(uintptr_t)(char PCH_LDS*)lds + wave * 1024;
    const char* kp = (const char*)uniform64((uint64_t)at<T>(A.k, w.k0, kvh));
    const char* vp = (const char*)uniform64((uint64_t)at<T>(A.v, w.k0, kvh));
    const auto load = [&](const char* p, int64_t token, int t, uint32_t to, const uint32_t (&off)[NL]) {
        const int left = w.len - t * KT, nr = (left < KT ? left : KT) - 1;
        const auto r = __builtin_amdgcn_make_buffer_rsrc((void*)(p + (int64_t)t * KT * token * 2), 0,
                                                         (nr * (int)token + A.dim) * 2, 0x00020000);
        load_lds<NW * 1024>(r, to, off);
    };
    const auto load_k = [&](int t) {
        if (t >= first) load(kp, A.k.token, t, base + (t & 1) * TB, ko);
    };
    const auto load_v = [&](int t) {
        if (t >= first) load(vp, A.v.token, t, base + (2 + (t & 1)) * TB, vo);
    };
    const auto arrived = [] { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    const auto keys = [&](int t) { return (const char PCH_LDS*)lds + (t & 1) * TB; };
    const auto values = [&](int t) { return (const char PCH_LDS*)lds + (2 + (t & 1)) * TB; };
    if (tiles > first) {
        load_k(tiles - 1);
        load_v(tiles - 1);
        load_k(tiles - 2);
    }
    Rows<T, DC> row;
    row.begin(A, w, kvh, group, mine + (lane & 31));
    // the keys [0, hi) are seen by rows of this wave; tiles below `whole` by every row of the workgroup: they need no mask
    const int sees = mine < R ? seen(w, mine + 31, group, A.causal) : 0;
    const int hi = keys_of<KT>(tiles, sees);
    const int every = seen(w, r0, group, A.causal) / KT;
    const int whole = clampi(every, first, tiles);

    // z: the scores of tile t, made while tile t + 1 was worked on
    v16f z[NK], zn[NK];
    int t = tiles - 1;
    settled();
    arrived();
    if (t >= first && t * KT < hi) W::scores(keys(t), row, z);
    for (; t >= whole; --t) {
        arrived();
        load_k(t - 2);
        load_v(t - 1);
        if (t > first && (t - 1) * KT < hi) W::scores(keys(t - 1), row, zn);
        if (t * KT < hi) {
            W::mask(row, t * KT, z);
            W::softmax(row, c, z);
            W::values(values(t), row, z);
        }
#pragma unroll
        for (int kb = 0; kb < NK; ++kb) z[kb] = zn[kb];
    }
    if ((A.causal || A.v.token < A.dim) && tiles_of<KT>(hi) > whole && W::broken(row)) W::repair(A, w, kvh, c, whole * KT, hi, KT, row);
    settled();
    float top = hi ? W::largest_of(z) : 0;
    // a step: tile t's weights and values, the scores of the one before; odd: t & 1
    const auto step = [&](int odd, v16f (&x)[NK], v16f (&y)[NK]) __attribute__((always_inline)) {
        arrived();
        load_k(t - 2);
        load_v(t - 1);
        if (!hi) return;
        W::grow(row, c, top);
        W::template scores<false>(keys(odd ^ 1), row, y);
        // the compiler's own pattern for products between LDS readings (256 dimensions 425 -> 405, prompt_long 1111 -> 1097)
        __builtin_amdgcn_iglp_opt(0);
        W::weigh(row, c, x);
        W::values(values(odd), row, x);
        top = W::largest_of(y);
    };
    const auto single = [&](int odd) __attribute__((always_inline)) {
        step(odd, z, zn);
#pragma unroll
        for (int kb = 0; kb < NK; ++kb) z[kb] = zn[kb];
        --t;
    };
    if constexpr (DC > 64) {
        // in pairs that begin at an even tile, z and zn taking turns: no copies, and the compiler knows the buffers (256
        // dimensions 427 -> 327 us, 192 333 -> 301, 96 127 -> 121, prompt_long 1067 -> 1048; but 64, causal, 177 -> 189)
        if (t > first && (t & 1)) single(1);
        while (t > first + 1) {
            step(0, z, zn);
            --t;
            step(1, zn, z);
            --t;
        }
        if (t > first) single(0);
    } else {
        for (; t > first; --t) {
            arrived();
            load_k(t - 2);
            load_v(t - 1);
            if (!hi) continue;
            W::grow(row, c, top);
            W::template scores<false>(keys(t - 1), row, zn);
            // the pattern for products between exponentials (8192 tokens x 16 heads 183 -> 173 us)
            __builtin_amdgcn_iglp_opt(2);
            W::weigh(row, c, z);
            W::values(values(t), row, z);
            top = W::largest_of(zn);
#pragma unroll
            for (int kb = 0; kb < NK; ++kb) z[kb] = zn[kb];
        }
    }
    if (t == first) {
        arrived();
        if (hi) {
            W::grow(row, c, top);
            W::weigh(row, c, z);
            W::values(values(t), row, z);
        }
    }
    W::finish(A, S, w, kvh, group, BM, wave * 32 + (lane & 31), row);
}

// ------------------------------------------------------------------------------------------------ few rows
// A workgroup of NW waves takes 32 rows (one token's heads of a group, mostly) and a part of their keys; the waves take its
// tiles of 32 keys in turn, each with LDS, statistics and sums of its own, and join at the end. What bounds it is the reading
// of the keys: 8 waves (4 above 128 dimensions: 128 KB either way) keep a tile of keys and one of values each on their way or
// in work, the next keys asked for as soon as the scores are made, the next values after the products (256 dimensions, 16
// caches of up to 8000: both after the products 40.3 us, so 37.2). 4 waves of two tiles each: 20 caches of up to 4000 56 -> 54
// us, 131072 keys 104.1 -> 103. One token, 64 heads on 8 key heads of 128, 131072 keys: 103 us, 5.2 TB/s (a large copy: 5.6);
// 48 caches of 89 to 8000 keys: 160 us, 5.1 TB/s. The 32 x 32 products leave most columns unused there; they take a tenth of
// the time of the reading.
template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

constexpr int AT_ONCE = 16;  // parts at most that a workgroup of few_k joins, all on their way at once

// two floats through the caches of this XCD to memory, and from there
__device__ __forceinline__ void through(float* p, float x, float y) {
    __hip_atomic_store((uint64_t*)p, (uint64_t)__float_as_uint(y) << 32 | __float_as_uint(x), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 past(const float* p) {
    const uint64_t v = __hip_atomic_load((const uint64_t*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

template <class T, int DP, int DC, int NW, bool TWICE>
__global__ void __launch_bounds__(64 * NW) few_k(AttentionArgs A, Split S, Group group) {
    constexpr int KT = 32, BM = 32, TB = KT * DP * 2, CPR = DP / 8, NL = KT * CPR / 64, PAD = DP + 4;
    using W = Wave<T, DP, DC, KT>;
    constexpr int JOIN = (NW * BM * PAD + NW * BM * 2) * 4, TILES = NW * 2 * TB;
    __shared__ __attribute__((aligned(1024))) char lds[JOIN > TILES ? JOIN : TILES];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int kvh = blockIdx.x;
    const Work w = locate<true, true>(A, S, blockIdx.z * gridDim.y + blockIdx.y, group.n, BM);
    if (!w.live) return;
    const int R = w.n * group.n, r0 = w.tile * BM;
    const float c = A.scale * 1.4426950408889634f;
    const int rn = R - r0 < BM ? R - r0 : BM;
    const int sees = seen(w, r0 + rn - 1, group, A.causal);
    const int all = tiles_of<KT>(sees);
    int first = 0, tiles = all;
    if (w.nc > 1) {
        first = (int)((int64_t)all * w.chunk / w.nc);
        tiles = (int)((int64_t)all * (w.chunk + 1) / w.nc);
    }
    const int hi = keys_of<KT>(tiles, sees);
    const int lo = seen(w, r0, group, A.causal);
    const int whole = lo / KT > first ? lo / KT : first;
    uint32_t ko[NL], vo[NL];
#pragma unroll
    for (int n = 0; n < NL; ++n) {
        const int p = n * 64 + lane, key = p / CPR, cp = p % CPR;
        const int ck = cp ^ Tile<DP>::kswz(key), cv = cp ^ Tile<DP>::vswz(key);
        ko[n] = ck * 8 < A.dim ? key * (uint32_t)A.k.token * 2 + ck * 16 : 0x7ffffff0u;
        vo[n] = cv * 8 < A.dim ? key * (uint32_t)A.v.token * 2 + cv * 16 : 0x7ffffff0u;
    }
    const uint32_t base = (uint32_t)(uintptr_t)(char PCH_LDS*)lds + wave * 2 * TB;
    const char* kp = (const char*)uniform64((uint64_t)at<T>(A.k, w.k0, kvh));
    const char* vp = (const char*)uniform64((uint64_t)at<T>(A.v, w.k0, kvh));
    const auto load = [&](const char* p, int64_t token, int t, uint32_t to, const uint32_t (&off)[NL]) {
        const int left = w.len - t * KT, nr = (left < KT ? left : KT) - 1;
        const auto r = __builtin_amdgcn_make_buffer_rsrc((void*)(p + (int64_t)t * KT * token * 2), 0,
                                                         (nr * (int)token + A.dim) * 2, 0x00020000);
        load_lds<1024>(r, to, off);
    };
    const auto load_k = [&](int t) { load(kp, A.k.token, t, base, ko); };
    const auto load_v = [&](int t) { load(vp, A.v.token, t, base + TB, vo); };
    // this wave's tiles, from the last of those that are `wave` mod NW after the first
    const int mine = tiles - first > wave ? (tiles - first - wave + NW - 1) / NW : 0;
    if (mine) {
        load_k(first + wave + (mine - 1) * NW);
        load_v(first + wave + (mine - 1) * NW);
    }
    Rows<T, DC> row;
    row.begin(A, w, kvh, group, r0 + (lane & 31));
    // TWICE: an infinite value times what the weights' rounding leaves, which has either sign or is zero, is no infinity of the
    // value's sign: there all of the wave's tiles are checked, at the end; else those that rows see in part, once they are done
    bool unchecked = TWICE;
    const auto mend = [&] {
        unchecked = false;
        if (W::broken(row)) {
            const int from = TWICE ? first : whole, skip = from - first > wave ? (from - first - wave + NW - 1) / NW : 0;
            W::repair(A, w, kvh, c, (uint32_t)(first + wave + skip * NW) * KT, hi, KT * NW, row);
            settled();
        }
    };
    const char PCH_LDS* const tl = (const char PCH_LDS*)lds + wave * 2 * TB;
    const auto read = [] { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };  // a tile's memory takes the next one
    settled();
    for (int u = mine - 1; u >= 0; --u) {
        const int t = first + wave + u * NW;
        wait_loads<NL>();
        v16f z[1];
        W::scores(tl, row, z);
        if (TWICE && u) {
            read();
            load_k(t - NW);
        }
        if (t >= whole) {
            W::mask(row, t * KT, z);
            unchecked |= (A.causal && lo < w.len) || A.v.token < A.dim;
        } else if (!TWICE && unchecked) {
            mend();
        }
        W::softmax(row, c, z);
        if (TWICE && u)
            wait_loads<NL>();
        else
            wait_loads<0>();
        W::template values<TWICE>(tl + TB, row, z);
        if (u) {
            read();
            if (!TWICE) load_k(t - NW);  // a prompt's, from L2: 2000 tokens x 12 heads of 64 26.4 us if asked for above, so 25.1
            load_v(t - NW);
        }
    }
    if (unchecked) mend();

    // the waves' sums joined: each scaled to the largest maximum, in the order of the waves
    float PCH_LDS* sh = (float PCH_LDS*)lds;
    float PCH_LDS* st = sh + NW * BM * PAD;
    const int cc = lane & 31, h = lane >> 5;
    const float l = row.l + other(row.l);
    __syncthreads();
    if (h == 0) st[wave * BM + cc] = row.m;
    __syncthreads();
    float m = -INFINITY;
#pragma unroll
    for (int x = 0; x < NW; ++x) m = fmaxf(m, st[x * BM + cc]);
    const float f = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(row.m - m);
    if (h == 0) st[NW * BM + wave * BM + cc] = l * f;
    if (cc < rn)
#pragma unroll
        for (int d = 0; d < DC / 32; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *(v4f PCH_LDS*)(sh + (wave * BM + cc) * PAD + 32 * d + 8 * g + 4 * h) =
                    v4f{row.o[d][4 * g] * f, row.o[d][4 * g + 1] * f, row.o[d][4 * g + 2] * f, row.o[d][4 * g + 3] * f};
    __syncthreads();
    const int slot = (w.slot + w.chunk) * A.kv_heads + kvh;
    const int q4 = A.dim >> 2;
    const auto store = [&](int r, int d, v4f o, float mr, float lr) {
        const int i = group.query(r0 + r), hd = kvh * group.n + (r0 + r - i * group.n);
        const float inv = lr == 0.0f ? 0.0f : 1.0f / lr;
        *(typename Mat<T>::v4*)(at<T>(A.out, w.q0 + i, hd) + d) = __builtin_convertvector(o * inv, typename Mat<T>::v4);
        if (A.lse && d == 0) A.lse[(int64_t)(w.q0 + i) * A.heads + hd] = logsum(mr, lr);
    };
    for (int x = threadIdx.x; x < rn * q4; x += 64 * NW) {
        const int r = x / q4, d = (x - r * q4) * 4;
        v4f o = *(const v4f PCH_LDS*)(sh + r * PAD + d);
        float lr = st[NW * BM + r], mr = st[r];
#pragma unroll
        for (int y = 1; y < NW; ++y) {
            o += *(const v4f PCH_LDS*)(sh + (y * BM + r) * PAD + d);
            lr += st[NW * BM + y * BM + r];
            mr = fmaxf(mr, st[y * BM + r]);
        }
        if (w.nc > 1) {
            float* const y = S.sums(slot, BM, A.dim) + r * A.dim + d;
            float* const ml = S.stats(slot, BM, A.dim) + r * 2;
            if (S.arrived) {
                through(y, o[0], o[1]);
                through(y + 2, o[2], o[3]);
                if (d == 0) through(ml, mr, lr);
            } else {
                *(v4f*)y = o;
                if (d == 0) *(float2*)ml = make_float2(mr, lr);
            }
        } else {
            store(r, d, o, mr, lr);
        }
    }
    if (w.nc == 1 || !S.arrived) return;

    // The part that is done last joins them all, in their order whatever order they were done in, where that is quicker than
    // join_k's launch. The sums go through the caches to memory that all XCDs see, and are there before the part is counted.
    __shared__ int last;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    int* const counter = S.arrived + w.slot / S.most * A.kv_heads + kvh;
    if (threadIdx.x == 0)
        last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == w.nc - 1;
    __syncthreads();
    if (!last) return;
    if (threadIdx.x == 0) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const int64_t step = (int64_t)A.kv_heads * BM;
    for (int x = threadIdx.x; x < rn * q4; x += 64 * NW) {
        const int r = x / q4, d = (x - r * q4) * 4;
        const float* y = S.sums(w.slot * A.kv_heads + kvh, BM, A.dim) + (int64_t)r * A.dim + d;
        const float* s2 = S.stats(w.slot * A.kv_heads + kvh, BM, A.dim) + r * 2;
        float mr = -INFINITY, lr = 0;
        v4f o = (v4f)0.0f;
        float2 a[AT_ONCE];
        v4f z[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            const int p = u < w.nc ? u : 0;
            const float* const g = y + p * step * A.dim;
            a[u] = past(s2 + p * step * 2);
            const float2 lo = past(g), hi = past(g + 2);
            z[u] = v4f{lo.x, lo.y, hi.x, hi.y};
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            if (u >= w.nc || a[u].y == 0.0f) continue;  // no such part, or no key in it
            const float mn = fmaxf(mr, a[u].x), f = __builtin_amdgcn_exp2f(mr - mn), g = __builtin_amdgcn_exp2f(a[u].x - mn);
            mr = mn;
            lr = lr * f + a[u].y * g;
            o = o * f + z[u] * g;
        }
        store(r, d, o, mr, lr);
    }
}

// ------------------------------------------------------------------------------------------------ parts of the keys joined
// 32 lanes of 4 dimensions to a row; PL lanes of parts (8 after few_k, whose parts may be many, 1 after rows_k, whose rows are),
// each merging every PL-th part, then the PL in their order; 8 / PL rows to a workgroup. Reading the parts is all there is to
// do, so they are read in parallel: one thread after the other through 128 parts took 120 us, 32 parts so take 5.5.
template <class T, int PL>
__global__ void __launch_bounds__(256) join_k(AttentionArgs A, Split S, Group group, int BM) {
    __shared__ v4f so[8][33];
    __shared__ float2 ss[8];
    const int blocks = BM * PL / 8, kvh = blockIdx.x / blocks, rb = blockIdx.x - kvh * blocks;
    const Work w = locate<false, false>(A, S, blockIdx.z * gridDim.y + blockIdx.y, group.n, BM);
    if (!w.live || w.nc == 1) return;
    const int q = threadIdx.x >> 5, pl = q % PL, dl = threadIdx.x & 31;
    const int R = w.n * group.n, r0 = w.tile * BM, rn = R - r0 < BM ? R - r0 : BM, r = rb * (8 / PL) + q / PL;
    const int64_t step = (int64_t)A.kv_heads * BM;
    for (int d0 = 0; d0 < A.dim; d0 += 128) {
        const int d = d0 + 4 * dl;
        const float* y = S.sums(w.slot * A.kv_heads + kvh, BM, A.dim) + (int64_t)r * A.dim + d;
        const float* st = S.stats(w.slot * A.kv_heads + kvh, BM, A.dim) + r * 2;
        float m = -INFINITY, l = 0;
        v4f o = (v4f)0.0f;
        for (int p0 = pl; r < rn && p0 < w.nc; p0 += 4 * PL) {  // four parts at a time on their way
            float2 x[4];
            v4f z[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int p = p0 + PL * u;
                const bool in = p < w.nc;
                x[u] = in ? *(const float2*)(st + p * step * 2) : make_float2(-INFINITY, 0);
                z[u] = in && d < A.dim ? *(const v4f*)(y + p * step * A.dim) : (v4f)0.0f;
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (x[u].y == 0.0f) continue;  // no key
                const float mn = fmaxf(m, x[u].x), a = __builtin_amdgcn_exp2f(m - mn), b = __builtin_amdgcn_exp2f(x[u].x - mn);
                m = mn;
                l = l * a + x[u].y * b;
                o = o * a + z[u] * b;
            }
        }
        if (PL > 1) {
            __syncthreads();
            so[q][dl] = o;
            if (dl == 0) ss[q] = make_float2(m, l);
            __syncthreads();
            if (pl == 0) {
                for (int p = 1; p < PL; ++p) m = fmaxf(m, ss[q + p].x);
                l = 0;
                o = (v4f)0.0f;
                for (int p = 0; p < PL; ++p) {
                    const float f = ss[q + p].y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ss[q + p].x - m);
                    l = fmaf(ss[q + p].y, f, l);
                    o += so[q + p][dl] * f;
                }
            }
        }
        if (pl || r >= rn || d >= A.dim) continue;
        const int i = group.query(r0 + r), hd = kvh * group.n + (r0 + r - i * group.n);
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        *(typename Mat<T>::v4*)(at<T>(A.out, w.q0 + i, hd) + d) = __builtin_convertvector(o * inv, typename Mat<T>::v4);
        if (A.lse && d == 0) A.lse[(int64_t)(w.q0 + i) * A.heads + hd] = logsum(m, l);
    }
}

// 0 and the arguments with their strides settled, or the error; the workspace, which its query does not read, apart
static int checked(const AttentionArgs* given, AttentionArgs* a) {
    if (!given) return -1;
    *a = *given;
    a->q = settled(a->q, a->tokens, a->heads, a->dim);
    a->out = settled(a->out, a->tokens, a->heads, a->dim);
    a->k = settled(a->k, a->kv_rows, a->kv_heads, a->dim);
    a->v = settled(a->v, a->kv_rows, a->kv_heads, a->dim);
    if (a->tokens < 0 || a->seqs < 0 || a->heads < 0 || a->kv_heads < 0 || a->kv_rows < 0 || a->max_q < 0 || a->max_k < 0)
        return -1;
    if (a->type != PCX_BF16 && a->type != PCX_F16) return -2;
    if (a->dim < 8 || a->dim > DMAX || a->dim % 8) return -2;
    if (!(a->scale > 0) || a->scale > 2.35e38f) return -1;  // times log2(e), as the kernels take it, finite
    if (a->heads && (a->kv_heads < 1 || a->heads % a->kv_heads)) return -1;
    if (a->seqs && a->tokens && a->heads && (!a->q_start || !a->k_start || !a->k_len)) return -1;
    if (!usable(a->q, a->tokens, a->heads) || !usable(a->out, a->tokens, a->heads) ||
        !usable(a->k, a->kv_rows, a->kv_heads) || !usable(a->v, a->kv_rows, a->kv_heads))
        return -1;
    for (const HeadsRef* r : {&a->q, &a->k, &a->v, &a->out})
        if ((uintptr_t)r->base % 16 || r->token % 8 || r->head % 8) return -2;
    if (!apart(a->out, a->tokens, a->heads, a->dim)) return -2;
    if (a->k.token > TOKEN_MAX || a->v.token > TOKEN_MAX) return -2;
    if ((int64_t)a->tokens * a->heads > ROWS_MAX) return -2;
    if (a->kv_heads > KV_HEADS_MAX) return -2;
    if (a->kv_heads && (int64_t)a->tokens * (a->heads / a->kv_heads) / 32 + a->seqs > ITEMS_MAX) return -2;
    return 0;
}

constexpr int COUNTERS = PCX_ATTENTION_COUNTERS;

// The kernel and the split of a call, by the lengths that the caller expects.
//  few_k: up to 32 rows of a key head; up to 128, whose tiles of 32 each read the keys, where those tiles are no more than the CUs
//  (rows_k and few_k in us: 16 queries x 32/8 heads over 8000 keys 24 and 19, 24 queries 24.8 and 21.5, 6 x 25 queries of 256
//  dimensions over 2000 41 and 30; but 30 x 16 queries over 1000 30 and 50) and above 64 rows the keys not many (24 queries over
//  16000 31 and 26, 32 over 50000 62 and 78); and at 64 dimensions, where two of its workgroups share a CU, prompts whose tiles
//  of 128 rows would not fill the chip (1024 tokens x 12 heads: 22 and 13; 2048: 34 and 25; at 128 dimensions, 500 tokens x 32:
//  16 and 22).
//  Splits: few_k to 256 workgroups, one a CU (131072 keys x 8 key heads: 192 or 256 workgroups 103 us, 384 114, 512 111) of at
//  least 384 keys, 48 a wave (4500 keys x 8 key heads: 256 a part 17.2 us, 384 14.4, the rest alike), 192 above 128 dimensions,
//  where the waves are 4 (2000 keys x 2 key heads of 256: 384 19.4, 192 16.6); rows_k to 512 of at least 512 keys (64 x 4
//  rows over 8000 keys: no split 166 us, 256 workgroups 32.5, 512 29.5; 2000 tokens x 32 heads: none 49, two parts 71).
struct Choice {
    bool few;       // few_k, else rows_k
    int BM;         // rows of a tile
    int64_t items;  // (sequence, tile) pairs at most
    int64_t base;   // workgroups there are likely to be without a split
    int most, size;
};
static uint64_t work_bytes(const AttentionArgs& a, const Choice& c) {
    return c.most > 1 ? COUNTERS * 4 + (uint64_t)c.items * c.most * a.kv_heads * c.BM * (a.dim + 2) * 4 : 0;
}

static Choice choose(const AttentionArgs& a) {
    const int group = a.heads / a.kv_heads;
    Choice c;
    const int64_t rows = (int64_t)a.max_q * group, tiles = (int64_t)a.tokens * group / 128 + a.seqs;
    const int64_t work = std::min<int64_t>((rows + 31) / 32, 5) * a.seqs * a.kv_heads;
    c.few = rows <= 32 || (rows <= 128 && work <= 256 && (rows <= 64 || work * a.max_k <= 3 << 18)) ||
            (a.dim <= 64 && tiles * a.kv_heads < 256);
    c.BM = c.few ? 32 : 128;
    c.items = (int64_t)a.tokens * group / c.BM + a.seqs;
    // the tiles there are likely to be, half a tile of each sequence's last one unused: one too many and a quarter of the chip may
    // idle (512 queries x 32/8 heads over 30000 keys: 3 parts 301 us, 4 fill it, 268)
    const int64_t spare = std::max<int64_t>((int64_t)a.seqs * c.BM / 2, c.BM - 1);
    const int64_t guess = std::min((rows + c.BM - 1) / c.BM * a.seqs, ((int64_t)a.tokens * group + spare) / c.BM);
    c.base = std::max<int64_t>(a.seqs, guess) * a.kv_heads;
    const int64_t want = c.few ? 256 : 512;
    const int shortest = !c.few ? 512 : a.dim > 128 ? 192 : 384;
    c.most = (int)std::max<int64_t>(1, std::min<int64_t>(want / std::max<int64_t>(c.base, 1), a.max_k / shortest));
    c.size = (int)(((int64_t)a.max_k + c.most - 1) / c.most);
    return c;
}

template <class T, int DP, int DC>
static int run_t(const AttentionArgs& a, hipStream_t s) {
    const int group = a.heads / a.kv_heads;
    Choice c = choose(a);
    while (c.most > 1 && (work_bytes(a, c) > (a.work ? a.work_bytes : 0) || c.items * c.most > ITEMS_MAX)) c.most = c.most / 2;
    if (c.most > 1) c.size = (int)(((int64_t)a.max_k + c.most - 1) / c.most);
    const Group g = {group, 1.0 / group};
    const int64_t tall = c.items * c.most, high = std::min<int64_t>(tall, 65535), deep = (tall + high - 1) / high;
    const dim3 grid((unsigned)a.kv_heads, (unsigned)high, (unsigned)deep);
    constexpr int NW = DP > 128 ? 4 : 8;
    // joined by the last part where its workgroup reads them all at once: 12 sequences x 2 parts 41 -> 35 us, 5 parts of 4 rows
    // 15.7 -> 14.9, but 52 parts of 8 rows 16.2 -> 20.4, 16 parts of 32 rows 22.6 -> 29.5
    const int64_t rows = std::min<int64_t>((int64_t)a.max_q * group, 32);
    const bool fused = c.few && c.most > 1 && c.most <= AT_ONCE && rows * a.dim <= 4 * 64 * NW && c.items * a.kv_heads <= COUNTERS;
    const Split S = {c.most, c.size, fused ? (int*)a.work : nullptr, (float*)a.work + COUNTERS, c.items * c.most * a.kv_heads};
    // the second product: not for the prompts of 64 dimensions that few_k takes, which it would make 13% slower; 4 waves for them
    // where there are workgroups for two a CU (1024 tokens x 12 heads: 8 waves 15.3 us, 4 13.4; 100 queries x 8 heads over
    // 4000 keys, 2 key heads: 16.1 and 18.8)
    const bool prompt = c.few && DP == 64 && (int64_t)a.max_q * group > 64;
    if (prompt && c.base > 256)
        hipLaunchKernelGGL((few_k<T, 64, 64, 4, false>), grid, dim3(256), 0, s, a, S, g);
    else if (prompt)
        hipLaunchKernelGGL((few_k<T, 64, 64, 8, false>), grid, dim3(512), 0, s, a, S, g);
    else if (c.few)
        hipLaunchKernelGGL((few_k<T, DP, DC, NW, true>), grid, dim3(64 * NW), 0, s, a, S, g);
    else
        hipLaunchKernelGGL((rows_k<T, DP, DC, 4>), grid, dim3(256), 0, s, a, S, g);
    if (c.most > 1 && !fused) {
        if (int e = launch_rc()) return e;
        const int64_t jh = std::min<int64_t>(c.items, 65535), jd = (c.items + jh - 1) / jh;
        const dim3 jg((unsigned)(a.kv_heads * (c.few ? c.BM : c.BM / 8)), (unsigned)jh, (unsigned)jd);
        if (c.few)
            hipLaunchKernelGGL((join_k<T, 8>), jg, dim3(256), 0, s, a, S, g, c.BM);
        else
            hipLaunchKernelGGL((join_k<T, 1>), jg, dim3(256), 0, s, a, S, g, c.BM);
    }
    return launch_rc();
}

template <class T>
static int run(const AttentionArgs& a, hipStream_t s) {
    if (a.dim <= 64) return run_t<T, 64, 64>(a, s);
    if (a.dim <= 96) return run_t<T, 128, 96>(a, s);
    if (a.dim <= 128) return run_t<T, 128, 128>(a, s);
    if (a.dim <= 192) return run_t<T, 256, 192>(a, s);
    return run_t<T, 256, 256>(a, s);
}

}  // namespace clear
}  // namespace pch

using namespace pch;
using namespace pch::clear;

extern "C" uint64_t pcx_attention_workspace(const AttentionArgs* args) {
    AttentionArgs a;
    if (checked(args, &a) || !a.tokens || !a.seqs || !a.heads) return 0;
    return work_bytes(a, choose(a));
}

extern "C" int pcx_attention(const AttentionArgs* args, pc_stream_t s) {
    AttentionArgs a;
    if (int e = checked(args, &a)) return e;
    if ((uintptr_t)a.work % 16) return -2;
    if (!a.tokens || !a.seqs || !a.heads) return 0;
    return a.type == PCX_BF16 ? run<bf16>(a, (hipStream_t)s) : run<f16>(a, (hipStream_t)s);
}
