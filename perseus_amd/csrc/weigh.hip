// What the queries of a call add to the weights of the keys that they see (pcx_key_weights).
//
// w_j = decay before_j + sum over the queries i that see j, and the heads h of the key's group, of exp(scale q_ih . k_j - lse_ih).
// The products z = q k^T leave a key to a lane: lane (c, h) (c = lane mod 32, h = lane / 32) has the scores of key c with the rows
// 8 i + 4 h + j (i, j < 4), so a key's sum grows inside its lane. Products, exponents and sums are f32; a sum grows by the sum of 16
// weights at a time. No two lanes add to the same word, so the sums have one order.
//
// weigh_k (prompts and chunks): the keys stay in registers, 64 to a wave; the rows go through LDS once for the four waves of a
// workgroup, the next tile asked for while this one is used; rows are split over workgroups and joined where the keys are few.
// weigh_few_k (up to 32 rows): the rows stay in registers and the keys are streamed.
//
// 8192 tokens x 32/8 heads of 128, causal, f16: 295 to 314 us by the card, 930 to 880 TFLOP/s (a 16384^3 product: 1280). Power
// takes a part of it: with queries or keys of zeros, whose products switch nothing, the same instructions take 234 us. Without the
// exponentials 292, without the products 149; what else keeps the products from the large product's rate is not measured (a
// 16-byte LDS reading serves two products here). One product after the other, then its exponentials: 329; deeper buffers, other
// interleavings, three waves a SIMD: within 2%.
#include <algorithm>

#include "tiles.h"

namespace pch {
namespace clear {

constexpr int rows_of(int dim) { return dim <= 128 ? 128 : 64; }  // rows of a tile: (query, head) pairs
constexpr int BK = 256;  // keys of a workgroup

struct Weigh {
    HeadsRef q, k, weights, before, places;
    const float* lse;
    const int32_t *q_start, *k_len, *next_place;
    const int64_t* k_start;  // null: pages
    PagesRef pages;
    float* work;  // [part][sequence][kv head][max_k] sums where rows are split
    int64_t kv_rows;
    int32_t tokens, seqs, heads, kv_heads, dim, causal, max_k;
    int32_t group, hb, qt, blocks;  // heads of a key head; of a tile, queries of a tile, tiles of a query's heads
    int32_t slots, parts;           // workgroups of a sequence's keys, parts of their rows
    uint32_t per_hb;                // 2^16 / hb, rounded up
    float scale, decay;
    // the query of a tile's row (exact for every lane of a workgroup: below 256)
    __device__ __forceinline__ int query(int x) const { return (int)(((uint32_t)x * per_hb) >> 16); }
};

// a sequence's queries and keys, within the buffers
struct Seq {
    int q0, n, len;
    int64_t k0;
    Seq() = default;
    // lane l's
    __device__ __forceinline__ Seq(const Seq& s, int l) {
        const auto of = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
        q0 = of(s.q0), n = of(s.n), len = of(s.len);
        k0 = (int64_t)((uint64_t)(uint32_t)of((int)((uint64_t)s.k0 >> 32)) << 32 | (uint32_t)of((int)s.k0));
    }
    __device__ __forceinline__ Seq(const Weigh& A, int b) {
        const auto clamp = [](int x, int hi) { return x < 0 ? 0 : x > hi ? hi : x; };
        q0 = clamp(A.q_start[b], A.tokens);
        n = clamp(A.q_start[b + 1], A.tokens) - q0;
        n = n < 0 ? 0 : n;
        len = A.k_len[b];
        len = len < 0 ? 0 : len;
        int64_t room;
        if (A.k_start) {
            k0 = A.k_start[b];
            room = k0 < 0 || k0 >= A.kv_rows ? 0 : A.kv_rows - k0;
        } else {
            k0 = (int64_t)b * A.pages.seq;
            room = A.pages.count ? (int64_t)A.pages.width << A.pages.log : 0;  // an empty pool has no rows
        }
        if (len > room) len = (int)room;
    }
    // the cache's row of key j; -1: on a page that the pool does not have
    __device__ __forceinline__ int64_t row(const Weigh& A, uint32_t j) const {
        if (A.k_start) return k0 + j;
        return A.pages.row(A.pages.table[k0 + (j >> A.pages.log)], j);
    }
    // the rows of two keys, their pages asked for at once
    __device__ __forceinline__ void two_rows(const Weigh& A, uint32_t j0, uint32_t j1, int64_t (&r)[2]) const {
        if (A.k_start) {
            r[0] = k0 + j0, r[1] = k0 + j1;
            return;
        }
        const int32_t* const table = A.pages.table + k0;
        const int page[2] = {table[j0 >> A.pages.log], table[j1 >> A.pages.log]};
        r[0] = A.pages.row(page[0], j0), r[1] = A.pages.row(page[1], j1);
    }
    // parts of the rows: lengths that the caller did not expect have no room for more than one
    __device__ __forceinline__ int parts(const Weigh& A) const { return len <= A.max_k ? A.parts : 1; }
};

// key j's new weight from the sum that the queries add (row: its row, before: its weight so far, if any); a query's own key
// begins at 0
__device__ __forceinline__ bool fresh(const Weigh& A, const Seq& S, uint32_t j) {
    return A.next_place && (int64_t)j >= (int64_t)S.len - S.n;
}
__device__ __forceinline__ float before(const Weigh& A, const Seq& S, int g, uint32_t j, int64_t row) {
    if (row < 0 || !A.before.base || A.decay == 0.0f || fresh(A, S, j)) return 0;
    return *((const float*)A.before.base + row * A.before.token + g * A.before.head);
}
__device__ __forceinline__ void put(const Weigh& A, const Seq& S, int b, int g, uint32_t j, int64_t row, float w) {
    if (row < 0) return;
    *((float*)A.weights.base + row * A.weights.token + g * A.weights.head) = w;
    if (A.places.base && fresh(A, S, j))
        *((int32_t*)A.places.base + row * A.places.token + g * A.places.head) = A.next_place[b] - (S.len - (int)j);
}
__device__ __forceinline__ float* partial(const Weigh& A, int part, int b, int g) {
    return A.work + (((int64_t)part * A.seqs + b) * A.kv_heads + g) * A.max_k;
}

template <class T, int DP, int DC>
__global__ void __launch_bounds__(256, 2) weigh_k(Weigh A) {
    typedef typename Mat<T>::v8 v8;
    typedef int v4i __attribute__((ext_vector_type(4)));
    constexpr int NW = 4, CPR = DP / 8, BR = rows_of(DP), TB = BR * DP * 2, NL = BR * CPR / (64 * NW), STEPS = DC / 16;
    __shared__ __attribute__((aligned(1024))) char lds[2 * TB];
    __shared__ __attribute__((aligned(16))) float nl[2][BR];  // less a row's log-sum-exp, in log2 units
    __shared__ __attribute__((aligned(16))) int lim[2][BR];   // the keys that it sees
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
    const int g = blockIdx.x, slot = A.parts == 1 ? blockIdx.y : blockIdx.y / A.parts, part = blockIdx.y - slot * A.parts;
    const int b = blockIdx.z;
    const Seq S(A, b);
    const int np = S.parts(A);
    if (part >= np || (int64_t)slot * BK >= S.len) return;
    const float c2 = A.scale * 1.4426950408889634f;
    const int tiles = (int)(((uint32_t)S.n + A.qt - 1) / A.qt) * A.blocks;
    // This lane's rows of a tile's loads (BR: none), and where they lie from the tile's first. In place of rows that the tile does not
    // have it takes the first again: of zeros, an infinity in a key would make a NaN where all rows' scores of it are -infinity.
    uint32_t off[NL], first[NL];
    int row_of[NL];
#pragma unroll
    for (int n = 0; n < NL; ++n) {
        const int p = (n * NW + wave) * 64 + lane, x = p / CPR, qi = A.query(x), hd = x - qi * A.hb;
        const int ch = (p % CPR) ^ Tile<DP>::kswz(x);
        row_of[n] = ch * 8 < A.dim && qi < A.qt ? x : BR;
        off[n] = ((uint32_t)qi * (uint32_t)A.q.token + (uint32_t)hd * (uint32_t)A.q.head) * 2 + ch * 16;
        first[n] = ch * 8 < A.dim ? ch * 16 : 0x7ffffff0u;  // past the dimensions: zeros
    }
    const int x0 = threadIdx.x, xq = A.query(x0), xh = x0 - xq * A.hb;  // the row whose log-sum-exp this lane of the first waves brings
    const uint32_t to = (uint32_t)(uintptr_t)(char PCH_LDS*)lds + wave * 1024;
    const T* const q = at<T>(A.q, S.q0, (int64_t)g * A.group);
    const float* const lse = A.lse + (int64_t)S.q0 * A.heads + (int64_t)g * A.group;

    // a tile's first query and head of the group, and its rows
    struct Rows {
        int i, hd, x;
    };
    const auto rows = [&](int t) {
        const int qb = A.blocks == 1 ? t : t / A.blocks, i = qb * A.qt, hd = A.blocks == 1 ? 0 : (t - qb * A.blocks) * A.hb;
        const int nq = S.n - i < A.qt ? S.n - i : A.qt, nh = A.group - hd < A.hb ? A.group - hd : A.hb;
        return Rows{i, hd, nq * nh};
    };
    const auto load = [&](int t, int buf) {
        const Rows r = rows(t);
        const char* p = (const char*)(q + (int64_t)r.i * A.q.token + (int64_t)r.hd * A.q.head);
        uint32_t own[NL];
#pragma unroll
        for (int n = 0; n < NL; ++n) own[n] = row_of[n] < r.x ? off[n] : first[n];
        load_lds<NW * 1024>(__builtin_amdgcn_make_buffer_rsrc((void*)uniform64((uint64_t)p), 0, 0x40000000, 0x00020000), to + buf * TB, own);
    };
    const auto ask = [&](int t) {
        const Rows r = rows(t);
        return x0 < r.x ? lse[(int64_t)(r.i + xq) * A.heads + r.hd + xh] : -INFINITY;
    };
    const auto bring = [&](int t, int buf, float x) {
        const Rows r = rows(t);
        nl[buf][x0] = x == -INFINITY ? x : x * -1.4426950408889634f;  // a row that sees no key adds nothing
        const int64_t sees = (int64_t)S.len - S.n + r.i + xq + 1;
        lim[buf][x0] = x0 >= r.x || sees < 0 ? 0 : (int)sees;
    };

    for (int64_t k0 = (int64_t)slot * BK; k0 < S.len; k0 += (int64_t)A.slots * BK) {
        // the tiles that see any of the keys, this part's of them; those from `whole` on see all of them
        const int64_t end = k0 + BK < S.len ? k0 + BK : S.len;
        const uint32_t i0 = A.causal && k0 + S.n > S.len ? k0 + S.n - S.len : 0, i1 = A.causal && end - 1 + S.n > S.len ? end - 1 + S.n - S.len : 0;
        const int begin = (int)(i0 / A.qt) * A.blocks, whole = (int)((i1 + A.qt - 1) / A.qt) * A.blocks;
        int t0 = begin, t1 = tiles;
        if (np > 1) {
            t0 = begin + (int)((double)(tiles - begin) * part / np);  // exact for the last part's end, one value for both neighbours
            t1 = begin + (int)((double)(tiles - begin) * (part + 1) / np);
        }
        float raw = 0;
        if (t0 < t1) {
            load(t0, 0);
            if (wave < BR / 64) raw = ask(t0);
        }
        // the keys of this wave, in registers; what the last tile has no key for is some row's, and not kept
        const uint32_t j = (uint32_t)k0 + wave * 64 + c, len = (uint32_t)S.len;
        int64_t key[2];
        S.two_rows(A, j < len ? j : len - 1, j + 32 < len ? j + 32 : len - 1, key);
        v8 kf[2][STEPS];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const T* x = at<T>(A.k, key[kb] < 0 ? 0 : key[kb], g);
#pragma unroll
            for (int s = 0; s < STEPS; ++s) kf[kb][s] = *(const v8*)(x + std::min(16 * s + 8 * h, A.dim - 8));
#pragma unroll
            for (int s = 0; s < STEPS; ++s)
                if (16 * s + 16 > A.dim && 16 * s + 8 * h >= A.dim) kf[kb][s] = (v8)(T)0.0f;
        }
        // after the loop lane (c, h) holds the sum of key j + 32 h
        const uint32_t mine = j + 32 * h;
        const int64_t row = h ? key[1] : key[0];
        const float old = np == 1 && mine < len ? before(A, S, g, mine, row) : 0;

        float acc[2] = {0, 0};
        const auto tile = [&](int buf, int x, bool masked) __attribute__((always_inline)) {
            const char PCH_LDS* const l = (const char PCH_LDS*)lds + buf * TB + c * DP * 2;
#pragma unroll
            for (int rb = 0; rb < BR / 32; ++rb) {
                if (x <= 32 * rb) break;
                v16f z[2];
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) z[kb] = (v16f)0.0f;
#pragma unroll
                for (int s = 0; s < STEPS; ++s) {
                    const v8 a = *(const v8 PCH_LDS*)(l + rb * 32 * DP * 2 + (((2 * s + h) ^ Tile<DP>::kswz(c)) << 4));
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb) z[kb] = Mat<T>::mul(a, kf[kb][s], z[kb]);
                }
                float part[2][4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const v4f m = *(const v4f*)&nl[buf][32 * rb + 8 * i + 4 * h];
                    v4i n;
                    if (masked) n = *(const v4i*)&lim[buf][32 * rb + 8 * i + 4 * h];
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb) {
                        float w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            w[e] = __builtin_amdgcn_exp2f(fmaf(z[kb][4 * i + e], c2, m[e]));
                            if (masked && j + 32 * kb >= (uint32_t)n[e]) w[e] = 0;
                        }
                        part[kb][i] = (w[0] + w[1]) + (w[2] + w[3]);
                    }
                }
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) acc[kb] += (part[kb][0] + part[kb][1]) + (part[kb][2] + part[kb][3]);
            }
        };
        // Rows that see all of the keys, up to 128 dimensions (above, the registers do not hold it): 32 rows' products beside the
        // exponentials of the 32 before, across tiles; the last ones' scores z1 and their rows' m1 wait for the next products (at the
        // beginning: none, weights of 0)
        v16f z0[2], z1[2];
        v4f m1[4];
        const auto products = [&](int buf, int rb, v16f (&z)[2]) __attribute__((always_inline)) {
            const char PCH_LDS* const l = (const char PCH_LDS*)lds + buf * TB + (32 * rb + c) * DP * 2;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) z[kb] = (v16f)0.0f;
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                const v8 a = *(const v8 PCH_LDS*)(l + (((2 * s + h) ^ Tile<DP>::kswz(c)) << 4));
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) z[kb] = Mat<T>::mul(a, kf[kb][s], z[kb]);
            }
        };
        const auto weights = [&](const v16f (&z)[2], const v4f (&m)[4]) __attribute__((always_inline)) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                float part[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = __builtin_amdgcn_exp2f(fmaf(z[kb][4 * i + e], c2, m[i][e]));
                    part[i] = (w[0] + w[1]) + (w[2] + w[3]);
                }
                acc[kb] += (part[0] + part[1]) + (part[2] + part[3]);
            }
        };
        const auto pair = [&](int buf, int rb) __attribute__((always_inline)) {
            products(buf, 2 * rb, z0);
            weights(z1, m1);
            __builtin_amdgcn_sched_barrier(0);
            v4f m0[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                m0[i] = *(const v4f*)&nl[buf][64 * rb + 8 * i + 4 * h];
                m1[i] = *(const v4f*)&nl[buf][64 * rb + 32 + 8 * i + 4 * h];
            }
            products(buf, 2 * rb + 1, z1);
            weights(z0, m0);
            __builtin_amdgcn_sched_barrier(0);
        };
        settled();
        if (t0 < t1) {
            if (wave < BR / 64) {
                bring(t0, 0, raw);
                if (t0 + 1 < t1) raw = ask(t0 + 1);
            }
            const auto step = [&](int t, bool masked) __attribute__((always_inline)) {
                const int buf = (t - t0) & 1;
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                if (t + 1 < t1) {
                    if (wave < BR / 64) {
                        bring(t + 1, buf ^ 1, raw);
                        if (t + 2 < t1) raw = ask(t + 2);
                    }
                    load(t + 1, buf ^ 1);
                }
                if constexpr (DP <= 128)
                    if (!masked) {
#pragma unroll
                        for (int rb = 0; rb < BR / 64; ++rb)
                            if (64 * rb < rows(t).x) pair(buf, rb);
                        return;
                    }
                tile(buf, rows(t).x, masked);
            };
            int t = t0;
            for (; t < t1 && t < whole; ++t) step(t, true);
#pragma unroll
            for (int i = 0; i < 4; ++i) z1[i & 1] = (v16f)0.0f, m1[i] = (v4f)-INFINITY;
            for (; t < t1; ++t) step(t, false);
            if constexpr (DP <= 128) weights(z1, m1);
        }
        const float both[2] = {acc[0] + other(acc[0]), acc[1] + other(acc[1])}, sum = h ? both[1] : both[0];
        if (mine < len) {
            if (np == 1)
                put(A, S, b, g, mine, row, fmaf(A.decay, old, sum));
            else
                partial(A, part, b, g)[mine] = sum;
        }
        if (k0 + (int64_t)A.slots * BK < S.len) __syncthreads();  // the next keys' first tile takes the memory of these keys' last
    }
}

// ------------------------------------------------------------------------------------------------ few rows
// 32 rows and fewer (tokens): the rows stay in registers, and each wave streams tiles of 32 keys past them through LDS of its own,
// two tiles of it: the next on its way while it works on this one. What bounds it is the reading of the keys. The tiles of all
// sequences are numbered in a row and cut into as many parts as the chip's waves hold of all key heads, so that lengths far apart leave
// none idle; neighbouring waves read neighbouring heads of the same keys (each its own part of all heads' tiles: 95 us, so 85: a
// row's heads lie together in memory). The sums of eight tiles wait in LDS until they are added to the weights before. A token each
// of 48 caches of 89 to 8000 keys x 8 heads of 128: 85 us, 5.0 TB/s (a large copy: 5.6).
constexpr int WINDOW = 8;

// the sequences' tiles of 32 keys, a lane per sequence, 64 sequences at a time
struct Tiles {
    int low, high;  // their inclusive sums within the 64, in two parts
    __device__ __forceinline__ int64_t upto(int lane) const {
        return ((int64_t)__builtin_amdgcn_readlane(high, lane) << 16) + __builtin_amdgcn_readlane(low, lane);
    }
    __device__ __forceinline__ int64_t mine() const { return ((int64_t)high << 16) + low; }
};
__device__ __forceinline__ Tiles tiles_of(const Seq& S, bool there) {
    const int t = there ? (int)(((uint32_t)S.len + 31) / 32) : 0;
    return {lane_sums(t & 0xffff), lane_sums(t >> 16)};
}

template <class T, int DP, int DC, int NW, bool PAGED>
__global__ void __launch_bounds__(64 * NW) weigh_few_k(Weigh A) {
    typedef typename Mat<T>::v8 v8;
    constexpr int STEPS = DC / 16, KT = 32, CPR = DP / 8, TB = KT * DP * 2, NL = KT * CPR / 64;
    __shared__ __attribute__((aligned(1024))) char lds[NW * 2 * TB];
    __shared__ __attribute__((aligned(16))) float gone[NW][32];  // less a row's log-sum-exp, in log2 units
    __shared__ __attribute__((aligned(16))) int limits[NW][32];  // the keys that it sees
    __shared__ float window[NW][WINDOW * KT];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
    float* const nl = gone[wave];
    int* const lim = limits[wave];
    float* const sums = window[wave];
    const float c2 = A.scale * 1.4426950408889634f;
    int64_t total = 0;
    for (int b0 = 0; b0 < A.seqs; b0 += 64) {
        const Tiles t = tiles_of(Seq(A, std::min(b0 + lane, A.seqs - 1)), b0 + lane < A.seqs);
        total += t.upto(63);
    }
    const int waves = gridDim.x * NW, parts = std::max(1, waves / A.kv_heads);
    uint32_t off[NL];
#pragma unroll
    for (int n = 0; n < NL; ++n) {
        const int p = n * 64 + lane, key = p / CPR, ch = (p % CPR) ^ Tile<DP>::kswz(key);
        off[n] = ch * 8 < A.dim ? (PAGED ? key % RUN : key) * (uint32_t)A.k.token * 2 + ch * 16 : 0x7ffffff0u;
    }
    const uint32_t base = (uint32_t)(uintptr_t)(char PCH_LDS*)lds + wave * 2 * TB;
    for (int unit = blockIdx.x * NW + wave; unit < parts * A.kv_heads; unit += waves) {
        const int part = unit / A.kv_heads, g = unit - part * A.kv_heads;
        int64_t now = (int64_t)((double)total * part / parts);
        const int64_t stop = (int64_t)((double)total * (part + 1) / parts);
        int b = -1;
        Seq S;
        int64_t start = 0, end = 0;  // the numbers of the sequence's tiles
        while (now < stop) {
            if (now >= end) {  // the sequence of this tile
                int64_t past = 0;
                b = -1;
                for (int b0 = 0; b0 < A.seqs && b < 0; b0 += 64) {
                    const Seq own(A, std::min(b0 + lane, A.seqs - 1));
                    const Tiles t = tiles_of(own, b0 + lane < A.seqs);
                    const uint64_t here = __ballot(past + t.mine() > now);
                    if (here) {
                        const int l = __builtin_ctzll(here);
                        b = b0 + l;
                        S = Seq(own, l);
                        start = past + (l ? t.upto(l - 1) : 0);
                        end = past + t.upto(l);
                    }
                    past += t.upto(63);
                }
                if (b < 0) return;
            }
            const int tiles = (int)(((uint32_t)S.len + KT - 1) / KT);
            const int first = (int)(now - start);
            const int last = (int)std::min<int64_t>(tiles, first + (stop - now));  // one past this wave's
            now += last - first;
            const char* const kp = (const char*)uniform64((uint64_t)at<T>(A.k, PAGED ? 0 : S.k0, g));
            page_t* const table = PAGED ? (page_t*)uniform64((uint64_t)(A.pages.table + S.k0)) : nullptr;
            Runs<NL, 1, CPR> pages;
            const auto load = [&](int t, int buf) __attribute__((always_inline)) {
                if constexpr (PAGED) {
                    pages.template load<KT, 1024>(A.pages, kp, (uint32_t)A.k.token * 2, A.dim, S.len, t, 0, base + buf * TB, off);
                } else {
                    const int left = S.len - t * KT, nr = (left < KT ? left : KT) - 1;
                    const auto r = __builtin_amdgcn_make_buffer_rsrc((void*)(kp + (int64_t)t * KT * A.k.token * 2), 0,
                                                                     (nr * (int)A.k.token + A.dim) * 2, 0x00020000);
                    load_lds<1024>(r, base + buf * TB, off);
                }
            };
            // 32 rows, query * group + head of the group; more only where more queries came than were expected: each 32 add to the last's
            const int64_t all = (int64_t)S.n * A.group;
            for (int64_t r0 = 0; r0 == 0 || r0 < all; r0 += 32) {
                if constexpr (PAGED) pages.template fetch<KT>(A.pages, table, S.len, first, 0);
                load(first, 0);
                if constexpr (PAGED) pages.template fetch<KT>(A.pages, table, S.len, first + 1, 0);
                const int R = all - r0 < 32 ? (int)(all - r0) : 32;
                const uint32_t r = (uint32_t)r0 + (c < R ? c : 0), i = A.group == 1 ? r : r / (uint32_t)A.group;
                const int64_t head = (int64_t)g * A.group + (r - i * A.group);
                v8 q[STEPS];
#pragma unroll
                for (int s = 0; s < STEPS; ++s) q[s] = (v8)(T)0.0f;
                if (R > 0) {  // (rows past the last are the first again, whose scores are no NaN where the first's are none)
                    const T* x = at<T>(A.q, S.q0 + (int64_t)i, head);
#pragma unroll
                    for (int s = 0; s < STEPS; ++s) q[s] = *(const v8*)(x + std::min(16 * s + 8 * h, A.dim - 8));
                }
                if (c < R) {
                    const float x2 = A.lse[(S.q0 + (int64_t)i) * A.heads + head];
                    nl[c] = x2 == -INFINITY ? x2 : x2 * -1.4426950408889634f;  // a row that sees no key adds nothing
                    const int64_t sees = A.causal ? (int64_t)S.len - S.n + i + 1 : S.len;
                    lim[c] = sees < 0 ? 0 : (int)sees;
                } else {
                    nl[c] = -INFINITY;
                    lim[c] = 0;
                }
#pragma unroll
                for (int s = 0; s < STEPS; ++s)
                    if (16 * s + 16 > A.dim && 16 * s + 8 * h >= A.dim) q[s] = (v8)(T)0.0f;
                // the weights before: on later rows, those that the earlier ones have written
                const bool begin = r0 == 0, kept = !begin || (A.before.base && A.decay != 0.0f), given = begin && kept;
                const float decay = begin ? A.decay : 1.0f;
                const float* const from = (const float*)(given ? A.before.base : A.weights.base) + g * (given ? A.before.head : A.weights.head);
                const int64_t step = given ? A.before.token : A.weights.token;
                // the keys that every row sees; of no row none, as zeros times an infinity in a key would make a NaN
                const int64_t whole = R < 1 ? 0 : A.causal && S.n > 1 ? (int64_t)S.len - S.n + 1 + (A.group == 1 ? r0 : r0 / A.group) : (int64_t)S.len + KT;
                settled();
                int buf = 0;
                for (int t0 = first; t0 < last; t0 += WINDOW) {
                    const int t1 = std::min(t0 + WINDOW, last);
                    for (int t = t0; t < t1; ++t, buf ^= 1) {
                        if (t + 1 < last) {
                            load(t + 1, buf ^ 1);
                            if constexpr (PAGED) pages.template fetch<KT>(A.pages, table, S.len, t + 2, 0);
                            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NL) : "memory");
                        } else {
                            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                        }
                        const char PCH_LDS* const l = (const char PCH_LDS*)lds + (wave * 2 + buf) * TB + c * DP * 2;
                        v16f z = (v16f)0.0f;
#pragma unroll
                        for (int s = 0; s < STEPS; ++s) z = Mat<T>::mul(q[s], *(const v8 PCH_LDS*)(l + (((2 * s + h) ^ Tile<DP>::kswz(c)) << 4)), z);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const v4f m = *(const v4f*)&nl[8 * e + 4 * h];
#pragma unroll
                            for (int u = 0; u < 4; ++u) z[4 * e + u] = __builtin_amdgcn_exp2f(fmaf(z[4 * e + u], c2, m[u]));
                        }
                        if ((int64_t)t * KT + KT > whole)
#pragma unroll
                            for (int e = 0; e < 16; ++e)
                                if ((int64_t)t * KT + c >= lim[8 * (e >> 2) + 4 * h + (e & 3)]) z[e] = 0;
                        float sum = ((z[0] + z[1]) + (z[2] + z[3])) + ((z[4] + z[5]) + (z[6] + z[7]));
                        sum += ((z[8] + z[9]) + (z[10] + z[11])) + ((z[12] + z[13]) + (z[14] + z[15]));
                        sum += other(sum);
                        if (h == 0) sums[(t - t0) * KT + c] = sum;
                    }
                    // loads on every path, all of them waited for here: one that the compiler took to be on its way at the next tile would
                    // make it wait there for that tile's keys too
                    const uint32_t j0 = (uint32_t)t0 * KT + lane, j1 = std::min((uint32_t)t1 * KT, (uint32_t)S.len);
                    int64_t row[WINDOW / 2];
                    float old[WINDOW / 2];
#pragma unroll
                    for (int e = 0; e < WINDOW / 2; ++e) row[e] = PAGED ? A.pages.table[S.k0 + (std::min(j0 + e * 64, j1 - 1) >> A.pages.log)] : 0;
#pragma unroll
                    for (int e = 0; e < WINDOW / 2; ++e) {
                        const uint32_t j = std::min(j0 + e * 64, j1 - 1);
                        row[e] = PAGED ? A.pages.row((int)row[e], j) : S.k0 + j;
                        old[e] = from[(row[e] < 0 ? 0 : row[e]) * step];
                    }
#pragma unroll
                    for (int e = 0; e < WINDOW / 2; ++e) asm volatile("" : "+v"(old[e]));
#pragma unroll
                    for (int e = 0; e < WINDOW / 2; ++e) {
                        const uint32_t j = j0 + e * 64;
                        const float sum = sums[e * 64 + lane];
                        if (j < j1) put(A, S, b, g, j, row[e], kept && !(begin && fresh(A, S, j)) ? fmaf(decay, old[e], sum) : sum);
                    }
                }
            }
        }
    }
}

// the parts of the rows joined, in their order: a lane a key
__global__ void __launch_bounds__(256) weigh_join_k(Weigh A) {
    const int g = blockIdx.y, b = blockIdx.z;
    const Seq S(A, b);
    const int np = S.parts(A);
    const uint32_t j = blockIdx.x * 256 + threadIdx.x;
    if (np == 1 || j >= (uint32_t)S.len) return;
    const int64_t row = S.row(A, j);
    float sum = 0;
    for (int p = 0; p < np; ++p) sum += partial(A, p, b, g)[j];
    put(A, S, b, g, j, row, fmaf(A.decay, before(A, S, g, j, row), sum));
}

static int checked(const KeyWeightsArgs* a, Weigh* w) {
    if (!a || a->tokens < 0 || a->seqs < 0 || a->heads < 0 || a->kv_heads < 0 || a->kv_rows < 0 || a->max_q < 0 || a->max_k < 0) return -1;
    if (a->type != PCX_BF16 && a->type != PCX_F16) return -2;
    if (a->dim < 8 || a->dim > 256 || a->dim % 8) return -2;
    if (!(a->scale > 0) || a->scale > 2.35e38f || !(a->decay >= 0) || a->decay > 3.4e38f) return -1;
    if (a->heads && (a->kv_heads < 1 || a->heads % a->kv_heads)) return -1;
    const bool any = a->seqs && a->kv_heads;
    if (any && (!a->q_start || !a->k_len || (a->tokens && a->heads && !a->lse))) return -1;
    if (a->cache.start && a->cache.pages) return -1;
    if (a->places.base && !a->next_place) return -1;
    *w = {};
    if (!a->cache.start)
        if (int e = pages_of(a->cache, any ? a->seqs : 0, a->kv_rows, &w->pages)) return any ? e : 0;
    if (!usable(a->q, a->tokens, a->heads) || !usable(a->k, a->kv_rows, a->kv_heads)) return -1;
    if (!usable(a->weights, any ? a->kv_rows : 0, a->kv_heads)) return -1;
    for (const HeadsRef* r : {&a->before, &a->places})
        if (r->token < 0 || r->head < 0) return -1;
    for (const HeadsRef* r : {&a->weights, &a->before, &a->places})
        if ((uintptr_t)r->base % 4) return -2;
    w->q = settled(a->q, a->tokens, a->heads, a->dim), w->k = settled(a->k, a->kv_rows, a->kv_heads, a->dim);
    w->weights = settled(a->weights, a->kv_rows, a->kv_heads, 1), w->before = settled(a->before, a->kv_rows, a->kv_heads, 1);
    w->places = settled(a->places, a->kv_rows, a->kv_heads, 1);
    for (const HeadsRef* r : {&w->q, &w->k})
        if ((uintptr_t)r->base % 16 || r->token % 8 || r->head % 8) return -2;
    if (!apart(w->weights, a->kv_rows, a->kv_heads, 1)) return -2;
    if ((int64_t)a->tokens * a->heads > 0x7fffffff - 127 || a->kv_heads > 65535 || a->seqs > 65535) return -2;
    w->k_start = a->cache.start;
    w->lse = a->lse, w->q_start = a->q_start, w->k_len = a->k_len, w->next_place = a->next_place;
    w->kv_rows = a->kv_rows;
    w->tokens = a->heads ? a->tokens : 0, w->seqs = a->seqs, w->heads = a->heads, w->kv_heads = a->kv_heads, w->dim = a->dim;
    w->causal = a->causal, w->max_k = a->max_k, w->scale = a->scale, w->decay = a->decay;
    w->group = a->heads && a->kv_heads ? a->heads / a->kv_heads : 1;
    const int BR = rows_of(w->dim);
    w->hb = w->group < BR ? w->group : BR;
    w->per_hb = (65536 + w->hb - 1) / w->hb;
    w->qt = BR / w->hb;
    w->blocks = (w->group + BR - 1) / BR;
    // a tile's offsets: below 2^30 bytes
    if (w->k.token > 1 << 22 || (!w->k_start && (w->k.token << w->pages.log) > PAGE_MAX)) return -2;
    if (w->q.token > (1 << 28) / w->qt || w->q.head > (1 << 28) / w->hb) return -2;
    return 0;
}

// How the rows are split: into workgroups for two a CU if they have a tile each, and up to 2048 where they have four tiles and more
// (8192 tokens x 32 heads: 1024 workgroups 329 us, 2048 317, 4096 323, 8192 354; as many parts of late keys, which few queries see,
// as leave all alike long: 351, a third round of them at its end). Where most queries see all keys of the one sequence, workgroups
// are alike by themselves, and two a CU are enough if they come out at that (4096 tokens x 32/8 heads, not causal: 2048 workgroups
// 142 us, 512 132; 2500 x 16/2 of 256 over 3200 131 and 85; 2048 queries x 16/4 heads over 32048 keys 262 and 252; but 384 of 1200
// queries over 12200 keys 87, where 768 take 79, and 8 sequences of up to 2000 keys 81, where it is 66). A workspace that is too
// small makes fewer.
static uint64_t bytes_of(const Weigh& w, int parts) {
    return parts > 1 ? PCX_ATTENTION_COUNTERS * 4 + (uint64_t)parts * w.seqs * w.kv_heads * w.max_k * 4 : 0;
}
static void choose(Weigh* w, int max_q, uint64_t room) {
    const int64_t tiles = ((int64_t)max_q + w->qt - 1) / w->qt * w->blocks;
    const int64_t keys = std::max<int64_t>(1, ((int64_t)w->max_k + BK - 1) / BK), pairs = (int64_t)w->seqs * w->kv_heads;
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(65535, (1 << 20) / pairs));
    w->slots = (int)std::min(keys, most);
    const int64_t base = (int64_t)w->slots * w->seqs * w->kv_heads;
    const bool alike = w->seqs == 1 && (!w->causal || w->max_k / 4 >= max_q) && base <= 512 && 512 % base <= 64;
    const int64_t most_of = std::min<int64_t>((alike ? 512 : 2048) / base, tiles / 4);
    w->parts = (int)std::max<int64_t>({1, std::min<int64_t>(512 / base, tiles), most_of});
    if (!w->max_k) w->parts = 1;  // no key is expected: there is nothing to join, and longer runs than expected are not split
    while (w->parts > 1 && (bytes_of(*w, w->parts) > room || w->slots * w->parts > 65535)) w->parts /= 2;
}

template <class T, bool PAGED>
static int run_few(const Weigh& w, hipStream_t s) {
    // as many waves as fit the chip, 160 KB of LDS each CU, and no more than tiles are expected
    const int wide = w.dim <= 64 ? 1024 : w.dim <= 128 ? 512 : 256;
    const int64_t tiles = (int64_t)w.seqs * w.kv_heads * std::max<int64_t>(1, ((int64_t)w.max_k + 31) / 32);
    const dim3 grid((unsigned)std::min<int64_t>(wide, (tiles + 3) / 4)), block(256);
    if (w.dim <= 64)
        hipLaunchKernelGGL((weigh_few_k<T, 64, 64, 4, PAGED>), grid, block, 0, s, w);
    else if (w.dim <= 96)
        hipLaunchKernelGGL((weigh_few_k<T, 128, 96, 4, PAGED>), grid, block, 0, s, w);
    else if (w.dim <= 128)
        hipLaunchKernelGGL((weigh_few_k<T, 128, 128, 4, PAGED>), grid, block, 0, s, w);
    else if (w.dim <= 192)
        hipLaunchKernelGGL((weigh_few_k<T, 256, 192, 4, PAGED>), grid, block, 0, s, w);
    else
        hipLaunchKernelGGL((weigh_few_k<T, 256, 256, 4, PAGED>), grid, block, 0, s, w);
    return launch_rc();
}

template <class T>
static int run(const Weigh& w, int max_q, hipStream_t s) {
    if ((int64_t)max_q * w.group <= 32) return w.k_start ? run_few<T, false>(w, s) : run_few<T, true>(w, s);
    const dim3 grid((unsigned)w.kv_heads, (unsigned)(w.slots * w.parts), (unsigned)w.seqs), block(256);
    if (w.dim <= 64)
        hipLaunchKernelGGL((weigh_k<T, 64, 64>), grid, block, 0, s, w);
    else if (w.dim <= 96)
        hipLaunchKernelGGL((weigh_k<T, 128, 96>), grid, block, 0, s, w);
    else if (w.dim <= 128)
        hipLaunchKernelGGL((weigh_k<T, 128, 128>), grid, block, 0, s, w);
    else if (w.dim <= 192)
        hipLaunchKernelGGL((weigh_k<T, 256, 192>), grid, block, 0, s, w);
    else
        hipLaunchKernelGGL((weigh_k<T, 256, 256>), grid, block, 0, s, w);
    if (int e = launch_rc()) return e;
    if (w.parts == 1) return 0;
    const dim3 keys((unsigned)((w.max_k + 255) / 256), (unsigned)w.kv_heads, (unsigned)w.seqs);
    hipLaunchKernelGGL(weigh_join_k, keys, block, 0, s, w);
    return launch_rc();
}

}  // namespace clear
}  // namespace pch

using namespace pch;
using namespace pch::clear;

extern "C" uint64_t pcx_key_weights_workspace(const KeyWeightsArgs* args) {
    Weigh w;
    if (checked(args, &w) || !args->seqs || !args->kv_heads) return 0;
    choose(&w, args->max_q, ~(uint64_t)0);
    return bytes_of(w, w.parts);
}

extern "C" int pcx_key_weights(const KeyWeightsArgs* args, pc_stream_t s) {
    Weigh w;
    if (int e = checked(args, &w)) return e;
    if ((uintptr_t)args->work % 16) return -2;
    if (!args->seqs || !args->kv_heads) return 0;
    choose(&w, args->max_q, args->work ? args->work_bytes : 0);
    w.work = (float*)args->work + PCX_ATTENTION_COUNTERS;
    return args->type == PCX_BF16 ? run<bf16>(w, args->max_q, (hipStream_t)s) : run<f16>(w, args->max_q, (hipStream_t)s);
}
