// What the clear side's matrix kernels share (attend.h, weigh.hip): the 32 x 32 products, tiles in LDS and their loads.
#pragma once
#include "clear.h"
#include "pages.h"

namespace pch {
namespace clear {

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

__device__ __forceinline__ uint64_t uniform64(uint64_t v) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return ((uint64_t)hi << 32) | lo;
}

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }


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
    static_assert(N == 1 || N == 2 || N % 4 == 0);
    if constexpr (N == 1) {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                     :
                     : "s"(lds), "v"(off[0]), "s"(r)
                     : "memory", "m0");
    } else if constexpr (N == 2) {
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

// ------------------------------------------------------------------------------------------------ keys in pages
// PAGED: a sequence's key j lies in row page[j / rows] rows + j mod rows of the pool (rows: a power of two, 16 at least; whole
// pages). Tiles of keys are loaded in runs of 16 rows, each in one page: a run has a buffer of its own, whose base the scalar unit
// makes while the wave works on the tile before, and the lanes' offsets are within the run. Page numbers are read by scalar loads
// a tile ahead, so that no tile waits for its table. A run past the sequence's end, or on a page that the pool does not have, is
// an empty buffer: it reads as zeros.
constexpr int64_t PAGE_MAX = 0x7fffffff;  // elements from a page to the next
typedef const int32_t __attribute__((address_space(4))) page_t;

template <int NL, int NW, int CPR>
struct Runs {
    static constexpr int PER = 64 / CPR;                                       // rows of a load
    static constexpr int E = PER * NW >= RUN ? NL : NL * PER * NW / RUN;       // runs that a wave takes a part of
    static constexpr int N = NL / E;                                           // its loads of one
    static_assert(E * N == NL && (N == 1 || N * PER * NW == RUN));
    int page[E];
    // the tile's run that the wave's loads e N .. e N + N - 1 take
    static __device__ __forceinline__ int run(int e, int wave) { return (e * N * NW + wave) * PER / RUN; }
    // page numbers of tile t, which may be past the last of the sequence's len keys
    template <int KT>
    __device__ __forceinline__ void fetch(const PagesRef& P, page_t* table, int len, int t, int wave) {
#pragma unroll
        for (int e = 0; e < E; ++e) page[e] = table[entry_of<KT>(t, run(e, wave) * RUN, P.log, len)];
    }
    // The scalar unit's instructions are in the way of the wave's others, so they are few for each run: what the tile alone decides
    // is made once (6 chunks of up to 512 queries over up to 6000 keys 169 -> 156 us; 161 where one run of rows takes 133, the same for
    // pages of 16 to 1024 rows in any order). Nearer to it came neither one buffer for a tile of one page (165), nor one for the whole pool with a
    // run as the scalar offset (33% behind), nor page numbers through LDS (157): what is left is not the number of these instructions
    // but the scalar registers, whose spilling takes vector registers that the products' addresses had. token: a row's distance in
    // bytes; a page's bytes stay in 32 bits.
    template <int KT, int STEP>
    __device__ __forceinline__ void load(const PagesRef& P, const char* base, uint32_t token, int dim, int len, int t, int wave,
                                         uint32_t lds, const uint32_t (&off)[NL]) const {
        const uint32_t row = (uint32_t)t * KT, mask = (1u << P.log) - 1, step = token << P.log;
        const int left = min(len - (int)row, KT), last = (left - 1) * (int)token + dim * 2, full = (RUN - 1) * (int)token + dim * 2;
        const char* const tile = base + (row & mask) * token;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint32_t at = run(e, wave) * RUN;
            const bool there = (uint32_t)page[e] < (uint32_t)P.count;
            int bytes = there ? max(min(last - (int)(at * token), full), 0) : 0;
            uint32_t id = there ? page[e] : 0;
            asm("" : "+s"(bytes), "+s"(id));  // selects, where the compiler would make a branch around each run
            const auto r = __builtin_amdgcn_make_buffer_rsrc((void*)(tile + (uint64_t)id * step + (at & mask) * token), 0, bytes, 0x00020000);
            uint32_t own[N];
#pragma unroll
            for (int n = 0; n < N; ++n) own[n] = off[e * N + n];
            load_lds<STEP>(r, lds + e * N * STEP, own);
        }
    }
};

}  // namespace clear
}  // namespace pch
