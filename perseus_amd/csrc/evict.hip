// Eviction from a cache: which keys leave (pcx_evict), and the rows that close the gaps (pcx_move_rows).
//
// Kept are the `keep` keys of a (sequence, key head) whose weights are largest, protected ones before all others, the lower key
// of two alike. The kept rows behind `keep` go to the gaps before it, both in rising order: as few moves as there are gaps, and
// none of them reads what another writes, so that they all run at once, in place.
#include <algorithm>
#include <type_traits>

#include "tiles.h"

namespace pch {
namespace clear {

// A cache's rows: row(b, j) of sequence b's key j, -1 on a page that the pool does not have
struct Rows {
    const int64_t* start;  // null: pages
    PagesRef p;
    int64_t rows;
    // where the sequence begins (pages: its table's first entry), and its length within the cache
    __device__ __forceinline__ int64_t begin(int b, int* len) const {
        int64_t at, room;
        if (start) {
            at = start[b];
            room = at < 0 || at >= rows ? 0 : rows - at;
        } else {
            at = (int64_t)b * p.seq;
            room = p.count ? (int64_t)p.width << p.log : 0;  // an empty pool has no rows
        }
        if (*len < 0) *len = 0;
        if (*len > room) *len = (int)room;
        return at;
    }
    __device__ __forceinline__ int64_t row(int64_t at, uint32_t j) const {
        if (start) return at + j;
        return p.row(p.table[at + (j >> p.log)], j);
    }
};

static int rows_of(const CacheRef& c, int64_t seqs, int64_t rows, Rows* r) {
    if (rows < 0 || (c.start && c.pages)) return -1;
    *r = {c.start, {}, rows};
    return c.start || !seqs ? 0 : pages_of(c, seqs, rows, &r->p);
}

// ------------------------------------------------------------------------------------------------ the choice
// A key's worth is a word of 64 bits, no two alike: the weight's bits in their order (protected keys above all), then the key's
// number from the top down. Kept are the keys from the keep-th largest word on. That word is found by its digits from the top: the
// words with the digits found so far are counted by their next one, 11 bits, in 2048 bins in LDS, until the bin that the last kept
// word is in is kept whole or holds few enough to rank each against all. Weights spread over orders of magnitude take one digit
// or two; a first digit is a quarter of an octave, so weights near each other take more.
//
// What bounds it are latencies: the loads of pages, weights and places, the counting's atomics, the barriers between. 528 keys x 12
// heads 5.3 us; 48 caches of 4160 keys x 8 heads 17; 65536 keys x 8 heads 31 in three launches. Three digits of every word in place of
// one and a ranking: 12, 32 and 168. Ranking up to 1024 words, 700 of them with as many: 32768 -> 8192 keys x 8 heads with the moves
// 69 us, 128 and fewer 37; up to 64: 48 caches of 4160 keys 27 us, so 23.
constexpr int WAVES = 16, THREADS = 64 * WAVES, BINS = 2048, RANKED = 128;
constexpr int SLICES = 16, PAIRS = 128, GATHERED = 8192, LONG = 16384;

struct Choice {
    HeadsRef weights, places;
    Rows cache;
    const int32_t *k_len, *next_place;
    int32_t *moves, *count, *kept_len;
    char* work;
    int32_t seqs, keep, recent, first, most, slices;
};

// a float's bits in an order of unsigned words: NaN 0, -infinity above it, +0 and -0 alike; +infinity is below PROTECTED
constexpr uint32_t PROTECTED = 0xffffffffu;
__device__ __forceinline__ uint32_t ordered(float w) {
    if (w != w) return 0;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t word(uint32_t key, uint32_t j) { return (uint64_t)key << 32 | ~j; }

struct Shared {
    uint32_t hist[BINS], sums[2][WAVES], found[3], n;
    uint64_t ranked[RANKED], least;
};

// the sum over the lanes of the waves before this one, and over all, of what each wave brings (the same to all its lanes)
__device__ __forceinline__ uint32_t waves_before(uint32_t (&sums)[WAVES], uint32_t mine, uint32_t* all) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (lane == 0) sums[wave] = mine;
    __syncthreads();
    const int in = lane_sums(lane < WAVES ? (int)sums[lane] : 0);
    *all = __builtin_amdgcn_readlane(in, WAVES - 1);
    return wave ? __builtin_amdgcn_readlane(in, wave - 1) : 0;
}

// the bin that the need-th largest is in: (bin, how many of its words are among them, its words), in found; x and y are the counts of
// bins BINS - 1 - 2 thread and the one below
__device__ __forceinline__ void find(Shared& S, uint32_t x, uint32_t y, uint32_t need) {
    const uint32_t in = lane_sums(x + y);
    uint32_t all;
    if (threadIdx.x < 3) S.found[threadIdx.x] = 0;  // of fewer words than that: none
    const uint32_t before = waves_before(S.sums[0], __builtin_amdgcn_readlane(in, 63), &all) + in - x - y;
    if (before < need && need <= before + x + y) {
        const bool second = need > before + x;
        S.found[0] = BINS - 1 - 2 * threadIdx.x - second;
        S.found[1] = need - before - (second ? x : 0);
        S.found[2] = second ? y : x;
    }
    __syncthreads();
}

// The need-th largest (need >= 1) of the words that each(f) calls f with, on the lanes that have them.
template <class Each>
__device__ __forceinline__ uint64_t select(Shared& S, uint32_t need, Each each) {
    uint64_t prefix = 0;
    for (int low = 53;; low = low == 32 ? 21 : low > 32 ? std::max(low - 11, 32) : std::max(low - 11, 0)) {
        const int bits = low == 32 || low == 0 ? 10 : 11, above = low + bits;
        S.hist[threadIdx.x] = S.hist[threadIdx.x + THREADS] = 0;
        if (threadIdx.x == 0) S.n = 0;
        __syncthreads();
        each([&](uint64_t w) {
            if (above == 64 || w >> above == prefix) atomicAdd(&S.hist[(w >> low) & ((1u << bits) - 1)], 1);
        });
        __syncthreads();
        find(S, S.hist[BINS - 1 - 2 * threadIdx.x], S.hist[BINS - 2 - 2 * threadIdx.x], need);
        prefix = prefix << bits | S.found[0];
        need = S.found[1];
        const uint32_t n = S.found[2];
        if (n == need || low == 0) return prefix << low;
        if (n > RANKED) continue;
        each([&](uint64_t w) {
            if (w >> low == prefix) S.ranked[atomicAdd(&S.n, 1) % RANKED] = w;  // (n of them, unless weights change meanwhile)
        });
        __syncthreads();
        if (threadIdx.x < n) {
            const uint64_t mine = S.ranked[threadIdx.x];
            uint32_t larger = 0;
            for (uint32_t i = 0; i < n; ++i) larger += S.ranked[i] > mine;
            if (larger == need - 1) S.least = mine;
        }
        __syncthreads();
        return S.least;
    }
}

// the words of a (sequence, key head)'s keys, E in the registers of each lane: a wave's lanes hold runs of 64 keys, its runs one
// after the other
template <int E, bool SMALL>
struct Words {
    const Choice& A;
    const int g, len;
    const int64_t at, next;
    uint32_t key[E];
    int from, seg;  // the chunk in registers: its first key, the keys of a wave's run
    static constexpr int CHUNK = THREADS * E;

    __device__ __forceinline__ Words(const Choice& a, int g, int b, int len, int64_t at)
        : A(a), g(g), len(len), at(at), next(a.next_place ? a.next_place[b] : len), from(0), seg(0) {}
    // this lane's first key (unsigned: past a run's last key a chunk has room for some beyond 2^31)
    __device__ __forceinline__ uint32_t first() const { return (uint32_t)from + (threadIdx.x >> 6) * (uint32_t)seg + (threadIdx.x & 63); }
    // The chunk of keys lo .. hi - 1, E loads of each kind on their way at once; those past the end read the last key again (loads under
    // a condition each: 48 caches of 4160 keys 25.6 us, so 23.7). SMALL: rows and their offsets in 32 bits.
    __device__ __forceinline__ void load(int lo, int hi) {
        typedef typename std::conditional<SMALL, uint32_t, int64_t>::type index;
        const char* const w = (const char*)A.weights.base + g * A.weights.head * 4;
        const char* const places = A.places.base ? (const char*)A.places.base + g * A.places.head * 4 : nullptr;
        const index w_row = (index)A.weights.token * 4, p_row = (index)A.places.token * 4;
        const bool paged = !A.cache.start;
        const int32_t* const table = A.cache.p.table + (paged ? at : 0);
        const uint32_t low = (1u << A.cache.p.log) - 1;
        from = lo;
        seg = 64 * ((hi - lo + THREADS - 1) / THREADS);
        if (lo >= hi) return;  // a slice of no key: there is no last one to read again
        int page[E], place[E];
        float x[E];
        const auto key_of = [&](int e) { return std::min(first() + e * 64, (uint32_t)hi - 1); };
        if (paged)
#pragma unroll
            for (int e = 0; e < E; ++e) page[e] = table[key_of(e) >> A.cache.p.log];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint32_t j = key_of(e);
            index row = (index)at + j;
            if (paged) {
                page[e] = (uint32_t)page[e] < (uint32_t)A.cache.p.count ? page[e] : -1;
                row = ((index)(page[e] < 0 ? 0 : page[e]) << A.cache.p.log) + (j & low);
            }
            x[e] = *(const float*)(w + row * w_row);
            if (places) place[e] = *(const int32_t*)(places + row * p_row);
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int64_t p = places ? place[e] : (int)key_of(e);
            key[e] = paged && page[e] < 0 ? 0 : p >= next - A.recent || p < A.first ? PROTECTED : ordered(x[e]);
        }
    }
    // f(e, j, word, whether there is one) in the order of e
    template <class F>
    __device__ __forceinline__ void each(int hi, F f) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (e * 64 >= seg) break;
            const uint32_t j = first() + e * 64;
            f(e, j, word(key[e], j), j < (uint32_t)hi);
        }
    }
    // f(word) for the keys lo .. hi - 1; loaded: they are in registers
    template <class F>
    __device__ __forceinline__ void all(int lo, int hi, bool loaded, F f) {
        for (int c = lo; c < hi; c += std::min(CHUNK, hi - c)) {
            const int end = c + std::min(CHUNK, hi - c);
            if (!loaded) load(c, end);
            each(end, [&](int, uint32_t, uint64_t w, bool in) {
                if (in) f(w);
            });
        }
    }
    // The moves of the keys lo .. hi - 1, least: the smallest word kept; movers, holes: of the keys before (each counts only from or to
    // `keep`), added to.
    __device__ __forceinline__ void emit(Shared& S, int lo, int hi, bool loaded, uint64_t least, int32_t* moves, uint32_t& movers, uint32_t& holes) {
        const uint64_t below = ((uint64_t)1 << (threadIdx.x & 63)) - 1;
        const uint32_t keep = A.keep;
        for (int c = lo; c < hi; c += std::min(CHUNK, hi - c)) {
            const int end = c + std::min(CHUNK, hi - c);
            if (!loaded) load(c, end);
            uint32_t m = 0, h = 0, all_m, all_h;
            each(end, [&](int, uint32_t j, uint64_t w, bool in) {
                m += __popcll(__ballot(in && w >= least && j >= keep));
                h += __popcll(__ballot(in && w < least && j < keep));
            });
            m = movers + waves_before(S.sums[0], m, &all_m);
            h = holes + waves_before(S.sums[1], h, &all_h);
            movers += all_m;
            holes += all_h;
            each(end, [&](int, uint32_t j, uint64_t w, bool in) {
                const bool mover = in && w >= least && j >= keep, hole = in && w < least && j < keep;
                const uint64_t ms = __ballot(mover), hs = __ballot(hole);
                const uint32_t to = m + __popcll(ms & below), gap = h + __popcll(hs & below);
                if (mover && to < (uint32_t)A.most) moves[2 * (int64_t)to] = j;
                if (hole && gap < (uint32_t)A.most) moves[2 * (int64_t)gap + 1] = j;
                m += __popcll(ms);
                h += __popcll(hs);
            });
            __syncthreads();
        }
    }
};

// a workgroup for each (sequence, key head)
template <int E, bool SMALL>
__global__ void __launch_bounds__(THREADS, E > 8 ? 4 : 8) evict_k(Choice A) {
    __shared__ Shared S;
    const int g = blockIdx.x, kv = gridDim.x;
    for (int b = blockIdx.y; b < A.seqs; b += gridDim.y) {
        int len = A.k_len[b];
        const int64_t at = A.cache.begin(b, &len), pair = (int64_t)b * kv + g;
        if (A.kept_len && g == 0 && threadIdx.x == 0) A.kept_len[b] = len < A.keep ? len : A.keep;
        uint32_t movers = 0, holes = 0;
        if (len > A.keep && A.keep) {
            Words<E, SMALL> W(A, g, b, len, at);
            const bool once = len <= W.CHUNK;
            if (once) W.load(0, len);
            const uint64_t least = select(S, A.keep, [&](auto f) { W.all(0, len, once, f); });
            W.emit(S, 0, len, once, least, A.moves + pair * A.most * 2, movers, holes);
        }
        if (threadIdx.x == 0) A.count[pair] = (int32_t)holes;
    }
}

// ------------------------------------------------------------------------------------------------ long caches
// Few pairs of long runs: 2 to 16 workgroups to each, a slice of its keys each (no slice on both sides of `keep`), in three launches. The
// slices' counts of the first digit; the words of the bin that is kept in part, gathered (8192 at most); the smallest word kept, and
// the slices' moves. Of more than 8192, as in long runs whose weights lie near each other, each workgroup goes through all words by
// itself. Weights exp(s normal), 8 heads, s of 2.5, 1, 0.5, 0.25 and 0.1: 65536 -> 16384 keys 28, 29, 34, 95 and 105 us; 131072 ->
// 32768 31, 34, 161, 166 and 187.
struct Pair {
    uint32_t hist[SLICES][BINS];
    uint64_t gathered[GATHERED];
    uint32_t found[3], kept[SLICES], some[SLICES];  // kept for certain, of the bin
};
static_assert(sizeof(Pair) % 8 == 0, "the gathered words stay aligned");

struct Slice {
    int lo, hi, before;  // its keys; the slices on its side of `keep` begin with this one
};
__device__ __forceinline__ Slice slice_of(int s, int slices, int len, int keep) {
    int left = (int)((int64_t)slices * keep / len);
    left = left < 1 ? 1 : left > slices - 1 ? slices - 1 : left;
    const auto cut = [](int n, int i, int of) { return (int)((int64_t)n * i / of); };
    if (s < left) return {cut(keep, s, left), cut(keep, s + 1, left), 0};
    const int n = len - keep, of = slices - left;
    return {keep + cut(n, s - left, of), keep + cut(n, s - left + 1, of), left};
}

template <int STAGE, bool SMALL>
__global__ void __launch_bounds__(THREADS) evict_long_k(Choice A) {
    __shared__ Shared S;
    constexpr int E = 8;
    const int g = blockIdx.x, kv = gridDim.x, s = blockIdx.y, b = blockIdx.z;
    int len = A.k_len[b];
    const int64_t at = A.cache.begin(b, &len), pair = (int64_t)b * kv + g;
    if (STAGE == 2 && A.kept_len && g == 0 && s == 0 && threadIdx.x == 0) A.kept_len[b] = len < A.keep ? len : A.keep;
    if (len <= A.keep || A.keep == 0) {
        if (STAGE == 2 && s == 0 && threadIdx.x == 0) A.count[pair] = 0;
        return;
    }
    Pair& P = ((Pair*)A.work)[pair];
    const Slice mine = slice_of(s, A.slices, len, A.keep);
    Words<E, SMALL> W(A, g, b, len, at);
    const bool once = mine.hi - mine.lo <= W.CHUNK;
    if (once) W.load(mine.lo, mine.hi);
    if constexpr (STAGE == 0) {
        S.hist[threadIdx.x] = S.hist[threadIdx.x + THREADS] = 0;
        __syncthreads();
        W.all(mine.lo, mine.hi, once, [&](uint64_t w) { atomicAdd(&S.hist[w >> 53], 1); });
        __syncthreads();
        *(uint2*)&P.hist[s][2 * threadIdx.x] = *(const uint2*)&S.hist[2 * threadIdx.x];
    } else if constexpr (STAGE == 1) {
        if (threadIdx.x == 0) S.n = 0;
        const int at2 = BINS - 2 - 2 * threadIdx.x;
        uint32_t x = 0, y = 0;
        uint2 own = make_uint2(0, 0);
#pragma unroll
        for (int i = 0; i < SLICES; ++i) {  // all asked for at once
            uint2 c = *(const uint2*)&P.hist[i < A.slices ? i : 0][at2];
            if (i >= A.slices) c = make_uint2(0, 0);
            x += c.y, y += c.x;
            if (i == s) own = c;
        }
        find(S, x, y, A.keep);
        const uint32_t bin = S.found[0], n = S.found[2];
        // the words of this slice above the bin, and of the slices before in it
        uint32_t above;
        const uint32_t sum = lane_sums((uint32_t)at2 > bin ? own.x + own.y : (uint32_t)at2 + 1 > bin ? own.y : 0);
        waves_before(S.sums[1], __builtin_amdgcn_readlane(sum, 63), &above);
        if (threadIdx.x == 0) {
            P.kept[s] = above;
            P.some[s] = P.hist[s][bin];
            if (s == 0) P.found[0] = bin, P.found[1] = S.found[1], P.found[2] = n;
        }
        if (n > GATHERED || n == S.found[1]) return;
        uint32_t to = 0;
        for (int i = 0; i < s; ++i) to += P.hist[i][bin];
        W.all(mine.lo, mine.hi, once, [&](uint64_t w) {
            if (w >> 53 == bin) P.gathered[(to + atomicAdd(&S.n, 1)) % GATHERED] = w;
        });
    } else {
        const uint32_t bin = P.found[0], need = P.found[1], n = P.found[2];
        uint64_t least = (uint64_t)bin << 53;
        uint32_t movers = 0, holes = 0, before = 0;  // kept of the slices on this side before this one
        if (n > GATHERED) {
            least = select(S, A.keep, [&](auto f) { W.all(0, len, false, f); });
            const int from = mine.before ? A.keep : 0;
            uint32_t kept = 0;
            W.all(from, mine.lo, false, [&](uint64_t w) { kept += w >= least; });
            if (once) W.load(mine.lo, mine.hi);
            __syncthreads();
            waves_before(S.sums[0], __builtin_amdgcn_readlane(lane_sums(kept), 63), &before);
            __syncthreads();
        } else {
            uint32_t some = 0, to = 0, from = 0;  // the bin's words before this slice, and before its side
            for (int i = 0; i < s; ++i) {
                if (i < mine.before) from += P.some[i];
                to += P.some[i];
                if (i >= mine.before) before += P.kept[i];
            }
            if (n == need) {
                before += to - from;
            } else {
                uint64_t w[GATHERED / THREADS];
#pragma unroll
                for (int i = 0; i < GATHERED / THREADS; ++i) w[i] = threadIdx.x + i * THREADS < n ? P.gathered[threadIdx.x + i * THREADS] : 0;
                least = select(S, need, [&](auto f) {
#pragma unroll
                    for (int i = 0; i < GATHERED / THREADS; ++i)
                        if (threadIdx.x + i * THREADS < n) f(w[i]);
                });
#pragma unroll
                for (int i = 0; i < GATHERED / THREADS; ++i) {
                    const uint32_t k = threadIdx.x + i * THREADS;
                    some += k >= from && k < to && w[i] >= least;
                }
                uint32_t all;
                waves_before(S.sums[1], __builtin_amdgcn_readlane(lane_sums(some), 63), &all);
                before += all;
                __syncthreads();
            }
        }
        if (mine.before)
            movers = before;
        else
            holes = mine.lo - before;
        W.emit(S, mine.lo, mine.hi, once, least, A.moves + pair * A.most * 2, movers, holes);
        if (!mine.before && mine.hi == A.keep && threadIdx.x == 0) A.count[pair] = (int32_t)holes;
    }
}

// ------------------------------------------------------------------------------------------------ the moves
struct Moves {
    HeadsRef t[4];
    int32_t size[4], row[4], unit[4];  // bytes of an element, of a row, of an access
    Rows cache;
    const int32_t *moves, *count;
    int32_t tensors, seqs, most, lanes_log, steps;
    __device__ __forceinline__ char* at(int i, int64_t r, int g, int o) const {
        return (char*)t[i].base + (r * t[i].token + g * t[i].head) * size[i] + o;
    }
    __device__ __forceinline__ uint4 load(int i, int64_t r, int g, int o) const {
        const char* p = at(i, r, g, o);
        if (unit[i] == 16) return *(const uint4*)p;
        return make_uint4(unit[i] == 4 ? *(const uint32_t*)p : *(const uint16_t*)p, 0, 0, 0);
    }
    __device__ __forceinline__ void store(int i, int64_t r, int g, int o, uint4 x) const {
        char* p = at(i, r, g, o);
        if (unit[i] == 16)
            *(uint4*)p = x;
        else if (unit[i] == 4)
            *(uint32_t*)p = x.x;
        else
            *(uint16_t*)p = (uint16_t)x.x;
    }
};

// A power of two of lanes takes a move, 16 bytes of a row each where addresses allow: the loads of all tensors, then the stores. It
// is bound by the memory, rows of one head a few hundred bytes each, out of order: 12480 moves x 8 heads of keys and values of 256
// bytes, weights and places, 104 MB: 23.5 us, 4.4 TB/s (a large copy: 5.6).
__global__ void __launch_bounds__(256) move_k(Moves A) {
    const int g = blockIdx.y, kv = gridDim.y, l = threadIdx.x & ((1 << A.lanes_log) - 1), each = 256 >> A.lanes_log;
    for (int b = blockIdx.z; b < A.seqs; b += gridDim.z) {
        const int64_t pair = (int64_t)b * kv + g;
        int n = A.count[pair];
        n = n < A.most ? n : A.most;
        for (int64_t i = (int64_t)blockIdx.x * each + (threadIdx.x >> A.lanes_log); i < n; i += (int64_t)gridDim.x * each) {
            const int2 m = *(const int2*)(A.moves + (pair * A.most + i) * 2);
            int room = 0x7fffffff;
            const int64_t at = A.cache.begin(b, &room);
            if ((uint32_t)m.x >= (uint32_t)room || (uint32_t)m.y >= (uint32_t)room) continue;
            const int64_t src = A.cache.row(at, m.x), dst = A.cache.row(at, m.y);
            if (src < 0 || dst < 0) continue;
            for (int s = 0; s < A.steps; ++s) {
                const int o = (s << A.lanes_log) + l;
                uint4 x[4];
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    if (t < A.tensors && o * A.unit[t] < A.row[t]) x[t] = A.load(t, src, g, o * A.unit[t]);
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    if (t < A.tensors && o * A.unit[t] < A.row[t]) A.store(t, dst, g, o * A.unit[t], x[t]);
            }
        }
    }
}

}  // namespace clear
}  // namespace pch

using namespace pch;
using namespace pch::clear;

template <bool SMALL>
static int run(const Choice& c, int kv_heads, int max_k, bool shared, hipStream_t s) {
    const dim3 block(THREADS);
    if (shared) {
        const dim3 grid(kv_heads, c.slices, c.seqs);
        hipLaunchKernelGGL((evict_long_k<0, SMALL>), grid, block, 0, s, c);
        if (int e = launch_rc()) return e;
        hipLaunchKernelGGL((evict_long_k<1, SMALL>), grid, block, 0, s, c);
        if (int e = launch_rc()) return e;
        hipLaunchKernelGGL((evict_long_k<2, SMALL>), grid, block, 0, s, c);
        return launch_rc();
    }
    const dim3 grid(kv_heads, std::min(c.seqs, 65535));
    // A word a lane where that is all (528 keys x 12 heads, five: 6.6 us, so 5.7). 5 take 64 registers, so that two workgroups share a
    // CU (48 caches of 4160 keys x 8 heads, registers not bounded: 32.4 us, so 25.6); of longer runs 16, read again for each digit
    // past 16384.
    if (max_k <= THREADS)
        hipLaunchKernelGGL((evict_k<1, SMALL>), grid, block, 0, s, c);
    else if (max_k <= 5 * THREADS)
        hipLaunchKernelGGL((evict_k<5, SMALL>), grid, block, 0, s, c);
    else
        hipLaunchKernelGGL((evict_k<16, SMALL>), grid, block, 0, s, c);
    return launch_rc();
}

// Few pairs of long runs, which a workgroup's registers do not hold: its own workgroups alone do not fill the chip. A workgroup each,
// and so, with the moves (8 heads of 64): 16384 keys 24 and 33 us, 20000 57 and 34, 65536 123 and 45; 16 caches of 20000 keys 127 and
// 113, 30 caches 198 and 210. 16 workgroups to each whatever the pairs: 8 caches of 16384 keys (128 dimensions) 157, a workgroup each 91.
static bool is_long(const EvictArgs& a) { return a.max_k > LONG && (int64_t)a.seqs * a.kv_heads <= PAIRS; }
static uint64_t work_bytes(const EvictArgs& a) { return PCX_ATTENTION_COUNTERS * 4 + (uint64_t)a.seqs * a.kv_heads * sizeof(Pair); }

extern "C" uint64_t pcx_evict_workspace(const EvictArgs* a) {
    return a && a->seqs > 0 && a->kv_heads > 0 && is_long(*a) ? work_bytes(*a) : 0;
}

extern "C" int pcx_evict(const EvictArgs* a, pc_stream_t s) {
    if (!a || a->seqs < 0 || a->kv_heads < 0 || a->keep < 0 || a->recent < 0 || a->first < 0 || a->most < 0 || a->max_k < 0) return -1;
    if ((int64_t)a->recent + a->first > a->keep) return -1;
    Choice c = {};
    if (int e = rows_of(a->cache, a->seqs, a->rows, &c.cache)) return e;
    const bool any = a->seqs && a->kv_heads;
    if (any && (!a->k_len || !a->count || (a->most && !a->moves) || a->kept_len == a->k_len)) return -1;
    if (!usable(a->weights, any ? a->rows : 0, a->kv_heads) || a->places.token < 0 || a->places.head < 0) return -1;
    if (((uintptr_t)a->weights.base | (uintptr_t)a->places.base) % 4 || (uintptr_t)a->work % 16 || a->kv_heads > 65535) return -2;
    if (!any) return 0;
    c.weights = settled(a->weights, a->rows, a->kv_heads, 1), c.places = settled(a->places, a->rows, a->kv_heads, 1);
    c.k_len = a->k_len, c.next_place = a->next_place;
    c.moves = a->moves, c.count = a->count, c.kept_len = a->kept_len;
    c.seqs = a->seqs, c.keep = a->keep, c.recent = a->recent, c.first = a->first, c.most = a->most;
    // offsets of 4-byte elements in 32 bits
    const bool small = a->rows < 0x3fffffff / std::max<int64_t>({1, c.weights.token, c.places.base ? c.places.token : 0});
    const bool shared = is_long(*a) && a->work && a->work_bytes >= work_bytes(*a);
    c.work = (char*)a->work + PCX_ATTENTION_COUNTERS * 4;
    c.slices = shared ? std::min(SLICES, 2 * PAIRS / (a->seqs * a->kv_heads)) : 1;
    return small ? run<true>(c, a->kv_heads, a->max_k, shared, (hipStream_t)s) : run<false>(c, a->kv_heads, a->max_k, shared, (hipStream_t)s);
}

extern "C" int pcx_move_rows(const MoveRowsArgs* a, pc_stream_t s) {
    if (!a || a->seqs < 0 || a->kv_heads < 0 || a->most < 0 || a->tensors < 0 || a->tensors > 4) return -1;
    Moves m = {};
    if (int e = rows_of(a->cache, a->seqs, a->rows, &m.cache)) return e;
    const bool any = a->seqs && a->kv_heads && a->most && a->tensors;
    if (any && (!a->moves || !a->count || (uintptr_t)a->moves % 8)) return -1;
    if (a->kv_heads > 65535) return -2;
    int units = 1;
    for (int i = 0; i < a->tensors; ++i) {
        if (!usable(a->t[i], any ? a->rows : 0, a->kv_heads)) return -1;
        if ((a->size[i] != 2 && a->size[i] != 4 && a->size[i] != 8) || a->dim[i] < 1 || a->dim[i] > 1 << 20) return -2;
        if (!apart(a->t[i], a->rows, a->kv_heads, a->dim[i])) return -2;
        m.t[i] = settled(a->t[i], a->rows, a->kv_heads, a->dim[i]);
        m.size[i] = a->size[i], m.row[i] = a->size[i] * a->dim[i];
        const uint64_t bits = (uintptr_t)m.t[i].base | (uint64_t)m.t[i].token * m.size[i] | (uint64_t)m.t[i].head * m.size[i] | m.row[i];
        if (bits % 2) return -2;
        m.unit[i] = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 2;
        if (m.row[i] / m.unit[i] > units) units = m.row[i] / m.unit[i];
    }
    if (!any) return 0;
    while (1 << m.lanes_log < units && m.lanes_log < 6) ++m.lanes_log;
    m.steps = (units + (1 << m.lanes_log) - 1) >> m.lanes_log;
    m.moves = a->moves, m.count = a->count;
    m.tensors = a->tensors, m.seqs = a->seqs, m.most = a->most;
    const int each = 256 >> m.lanes_log, deep = a->seqs < 65535 ? a->seqs : 65535;
    // a workgroup for each `each` moves that there may be; where that is many, so many in all, and each goes on to more
    const int64_t wide = ((int64_t)a->most + each - 1) / each, most = 65536 / ((int64_t)a->kv_heads * deep) + 1;
    const dim3 grid((unsigned)(wide < most ? wide : most), a->kv_heads, deep);
    hipLaunchKernelGGL(move_k, grid, dim3(256), 0, (hipStream_t)s, m);
    return launch_rc();
}
