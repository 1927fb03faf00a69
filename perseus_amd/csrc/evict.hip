// Eviction from a cache: which keys leave (pcx_evict), and the rows that close the gaps (pcx_move_rows).
//
// Kept are the `keep` keys of a (sequence, key head) whose weights are largest, protected ones before all others, the lower key
// of two alike. The kept rows behind `keep` go to the gaps before it, both in rising order: as few moves as there are gaps, and
// none of them reads what another writes, so that they all run at once, in place.
#include "clear.h"

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
            room = (int64_t)p.width << p.log;
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
struct Choice {
    HeadsRef weights, places;
    Rows cache;
    const int32_t *k_len, *next_place;
    int32_t *moves, *count, *kept_len;
    int32_t seqs, keep, recent, first, most;
};

// a float's bits in an order of unsigned words: NaN 0, -infinity above it, +0 and -0 alike; +infinity is below PROTECTED
constexpr uint32_t PROTECTED = 0xffffffffu;
__device__ __forceinline__ uint32_t ordered(float w) {
    if (w != w) return 0;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int WAVES = 16, BINS = 2048;

// the sum over the lanes below and this one
__device__ __forceinline__ uint32_t upto(uint32_t x) {
    const int lane = threadIdx.x & 63;
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t y = __shfl_up(x, d);
        if (lane >= d) x += y;
    }
    return x;
}

// A workgroup takes a (sequence, key head). The smallest word kept is found digit by digit, 11, 11 and 10 bits from the top, by
// counting the words with the digits found so far in 2048 bins; then ranks are counted by ballots, a wave a run of keys. A chunk
// of 1024 E words stays in registers; of more keys than that the words are made again for each digit.
struct Counts {
    uint32_t hist[BINS], sums[3][WAVES], found[2];
};

template <int E>
__device__ __forceinline__ void choose(const Choice& A, int b, Counts& S) {
    constexpr int CHUNK = 64 * WAVES * E, BATCH = E > 16 ? 8 : 16;  // rows whose loads are on their way at once
    auto& hist = S.hist;
    auto& sums = S.sums;
    auto& found = S.found;
    const int g = blockIdx.x, kv = gridDim.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int len = A.k_len[b];
    const int64_t at = A.cache.begin(b, &len);
    int32_t* const count = A.count + (int64_t)b * kv + g;
    if (A.kept_len && g == 0 && threadIdx.x == 0) A.kept_len[b] = len < A.keep ? len : A.keep;
    if (len <= A.keep || A.keep == 0) {
        if (threadIdx.x == 0) *count = 0;
        return;
    }
    const int64_t next = A.next_place ? A.next_place[b] : len;
    const float* const w = (const float*)A.weights.base + g * A.weights.head;
    const int32_t* const places = A.places.base ? (const int32_t*)A.places.base + g * A.places.head : nullptr;
    uint32_t key[E];
    int c0, seg;  // the chunk in registers: its first key, the keys of a wave's run
    const auto load = [&](int from) {
        c0 = from;
        const int n = len - from < CHUNK ? len - from : CHUNK;
        seg = 64 * ((n + 64 * WAVES - 1) / (64 * WAVES));
#pragma unroll
        for (int e0 = 0; e0 < E; e0 += BATCH) {
            if (e0 * 64 >= seg) break;
            int64_t row[BATCH];
#pragma unroll
            for (int e = 0; e < BATCH; ++e) {
                const int j = from + wave * seg + (e0 + e) * 64 + lane;
                row[e] = (e0 + e) * 64 < seg && j < len ? A.cache.row(at, j) : -1;
            }
            float x[BATCH];
            int place[BATCH];
#pragma unroll
            for (int e = 0; e < BATCH; ++e) {
                x[e] = row[e] < 0 ? 0 : w[row[e] * A.weights.token];
                place[e] = row[e] < 0 ? 0 : places ? places[row[e] * A.places.token] : from + wave * seg + (e0 + e) * 64 + lane;
            }
#pragma unroll
            for (int e = 0; e < BATCH; ++e)
                key[e0 + e] = row[e] < 0 ? 0 : place[e] >= next - A.recent || place[e] < A.first ? PROTECTED : ordered(x[e]);
        }
    };
    // f(e, j, key) for the chunk's keys of this lane, in the order of e
    const auto each = [&](auto f) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (e * 64 >= seg) break;
            const int j = c0 + wave * seg + e * 64 + lane;
            f(e, j, key[e], j < len);
        }
    };
    const bool once = len <= CHUNK;
    if (once) load(0);
    uint32_t prefix = 0, need = A.keep;
    for (int p = 0; p < 3; ++p) {
        const int low = p == 0 ? 21 : p == 1 ? 10 : 0, above = p == 0 ? 0 : p == 1 ? 21 : 10;
        const uint32_t mask = p == 2 ? 1023 : 2047;
        hist[threadIdx.x] = hist[threadIdx.x + 1024] = 0;
        __syncthreads();
        for (int from = 0; from < len; from += CHUNK) {
            if (!once) load(from);
            each([&](int, int, uint32_t k, bool in) {
                if (in && (p == 0 || k >> above == prefix)) atomicAdd(&hist[(k >> low) & mask], 1);
            });
        }
        __syncthreads();
        // bins from the top, two to a thread: the one where the words kept begin
        const uint32_t x = hist[BINS - 1 - 2 * threadIdx.x], y = hist[BINS - 2 - 2 * threadIdx.x], in = upto(x + y);
        if (lane == 63) sums[0][wave] = in;
        __syncthreads();
        uint32_t before = in - x - y;
        for (int v = 0; v < wave; ++v) before += sums[0][v];
        if (before < need && need <= before + x + y) {
            const bool second = need > before + x;
            found[0] = BINS - 1 - 2 * threadIdx.x - second;
            found[1] = need - before - (second ? x : 0);
        }
        __syncthreads();
        prefix = p == 0 ? found[0] : prefix << (p == 1 ? 11 : 10) | found[0];
        need = found[1];  // of the words with these digits
    }
    // prefix: the smallest word kept; need: how many of those alike stay, the lowest
    const uint64_t below = ((uint64_t)1 << lane) - 1;
    int32_t* const moves = A.moves + ((int64_t)b * kv + g) * A.most * 2;
    uint32_t ties = 0, movers = 0, holes = 0;  // of the chunks before
    for (int from = 0; from < len; from += CHUNK) {
        if (!once) load(from);
        uint32_t n = 0;
        each([&](int, int, uint32_t k, bool in) { n += __popcll(__ballot(in && k == prefix)); });
        if (lane == 0) sums[0][wave] = n;
        __syncthreads();
        uint32_t tie = ties, m = 0, h = 0;
        for (int v = 0; v < WAVES; ++v) {
            tie += v < wave ? sums[0][v] : 0;
            ties += sums[0][v];
        }
        uint64_t kept = 0;
        each([&](int e, int j, uint32_t k, bool in) {
            const uint64_t alike = __ballot(in && k == prefix);
            const bool stays = in && (k > prefix || (k == prefix && tie + __popcll(alike & below) < need));
            tie += __popcll(alike);
            kept |= (uint64_t)stays << e;
            m += __popcll(__ballot(stays && j >= A.keep));
            h += __popcll(__ballot(in && !stays && j < A.keep));
        });
        if (lane == 0) sums[1][wave] = m, sums[2][wave] = h;
        __syncthreads();
        m = movers, h = holes;
        for (int v = 0; v < WAVES; ++v) {
            m += v < wave ? sums[1][v] : 0;
            h += v < wave ? sums[2][v] : 0;
            movers += sums[1][v];
            holes += sums[2][v];
        }
        each([&](int e, int j, uint32_t, bool in) {
            const bool stays = kept >> e & 1;
            const uint64_t mover = __ballot(stays && j >= A.keep), hole = __ballot(in && !stays && j < A.keep);
            const uint32_t to = m + __popcll(mover & below), gap = h + __popcll(hole & below);
            if (stays && j >= A.keep && to < (uint32_t)A.most) moves[2 * (int64_t)to] = j;
            if (in && !stays && j < A.keep && gap < (uint32_t)A.most) moves[2 * (int64_t)gap + 1] = j;
            m += __popcll(mover);
            h += __popcll(hole);
        });
        __syncthreads();
    }
    if (threadIdx.x == 0) *count = (int32_t)holes;
}

template <int E>
__global__ void __launch_bounds__(64 * WAVES) evict_k(Choice A) {
    __shared__ Counts S;
    for (int b = blockIdx.y; b < A.seqs; b += gridDim.y) choose<E>(A, b, S);
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

// A power of two of lanes takes a move, 16 bytes of a row each where addresses allow: the loads of all tensors, then the stores.
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

extern "C" int pcx_evict(const EvictArgs* a, pc_stream_t s) {
    if (!a || a->seqs < 0 || a->kv_heads < 0 || a->keep < 0 || a->recent < 0 || a->first < 0 || a->most < 0 || a->max_k < 0) return -1;
    if ((int64_t)a->recent + a->first > a->keep) return -1;
    Choice c = {};
    if (int e = rows_of(a->cache, a->seqs, a->rows, &c.cache)) return e;
    const bool any = a->seqs && a->kv_heads;
    if (any && (!a->k_len || !a->count || (a->most && !a->moves) || a->kept_len == a->k_len)) return -1;
    if (!usable(a->weights, any ? a->rows : 0, a->kv_heads) || a->places.token < 0 || a->places.head < 0) return -1;
    if (((uintptr_t)a->weights.base | (uintptr_t)a->places.base) % 4 || a->kv_heads > 65535) return -2;
    if (!any) return 0;
    c.weights = settled(a->weights, a->rows, a->kv_heads, 1), c.places = settled(a->places, a->rows, a->kv_heads, 1);
    c.k_len = a->k_len, c.next_place = a->next_place;
    c.moves = a->moves, c.count = a->count, c.kept_len = a->kept_len;
    c.seqs = a->seqs, c.keep = a->keep, c.recent = a->recent, c.first = a->first, c.most = a->most;
    const dim3 grid(a->kv_heads, a->seqs < 65535 ? a->seqs : 65535);
    hipLaunchKernelGGL((evict_k<16>), grid, dim3(64 * WAVES), 0, (hipStream_t)s, c);
    return launch_rc();
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
