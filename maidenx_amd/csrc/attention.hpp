// Causal attention over packed sequences with grouped heads and an optional learned relative position bias, forward and
// backward, in tiles that never leave the chip.
//
//   S_ij = scale * q_i . k_j + table[bucket(i - j)][h]     j <= i, both in one sequence [offsets[s], offsets[s + 1])
//   o_i  = sum_j P_ij v_j,  P_ij = exp(S_ij - lse_i),  lse_i = ln sum_j exp S_ij
//   dP_ij = do_i . v_j;  D_i = do_i . o_i = sum_j P_ij dP_ij;  dS_ij = P_ij (dP_ij - D_i)
//   dq_i = scale sum_j dS_ij k_j;  dk_j = scale sum_i dS_ij q_i;  dv_j = sum_i P_ij do_i   (sums over the heads of a group too)
//   dtable[b][h] = sum of dS_ij over the pairs with bucket(i - j) = b
//
// Layout of the products.  All of them are 32 x 32 tiles of the matrix cores, with the fragment of a lane l (half = l / 32)
//   operand:  row l % 32, eight terms of the sum starting at 8 * half       result:  column l % 32, rows (r % 4) + 8 (r / 4) + 4 half
// S is formed with the index that the next product does NOT sum over in the columns: S^T = K Q^T where o and dq sum over
// keys, S = Q K^T where dk and dv sum over queries.  A lane then holds, for its own column, eight values of every half of
// a 32-row tile, which IS the right operand of the next product once both operands agree on the order of the terms: the
// left operand (v, k, do, q with the summed index in the rows) is read from LDS transposed, in that order.  So P and dS
// never travel between lanes, and the softmax statistics of a query are one register of its lane (plus one exchange of halves).
//
// Tiles are laid over the packed tokens, not over sequences: a row knows its sequence's first token, tiles that no mask
// touches skip it, and a batch of short sequences fills its tiles.
//
// Rounding: scores, statistics and every accumulator are f32.  P and dS are rounded to the tensors' type where they become an
// operand of the matrix cores (bf16 and f16; f32 tensors keep f32 there): a term t of a sum is then off by u |t| at most (u = 2^-8, 2^-11),
// the sum by u times the sum of the |t|, and by about u times the root of the sum of their squares, the roundings being independent; the
// result's own rounding is u times the sum.  Against 64 bits that makes 1.3 times (output) and 1.5 times (gradients) the error
// of the same formulas with P and dS in f32.  What f16 cannot hold of dS is scaled by powers of two (AttnLift).
#pragma once
#include <cmath>
#include <cstring>
#include <type_traits>

#include "attention_walk.hpp"
#include "mxh.hpp"

namespace mxh {

constexpr int ATTN_MAX_DIM = 128;
constexpr int ATTN_MAX_BUCKETS = 256;
constexpr int ATTN_MAX_DISTANCE = 4096;
constexpr int ATTN_THREADS = 256, ATTN_WAVES = ATTN_THREADS / WAVE;
constexpr int ATTN_ROWS = 128;              // rows (of queries, or of keys in the backward pass for keys) that a block owns: 32 a wave
constexpr float ATTN_LOG2E = 1.4426950408889634f, ATTN_LN2 = 0.6931471805599453f;

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef float f32x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));

template <class E>
struct AttnView {              // one [tokens, heads, dim] operand
    const E* p;
    int64_t token, head, elem; // strides in elements
    int vec;                   // rows can be read in 16-byte pieces
};
template <class E>
struct AttnArgs {
    AttnView<E> q, k, v, o, go;
    const int32_t* offsets;
    const E* table;            // [buckets, heads], null: no bias
    int32_t tokens, heads, group, dim, sequences;
    int32_t buckets, exact_to, max_distance;
    float scale, scale_abs, scale_log2;   // scale_log2 = |scale| * log2(e); the sign goes into an operand
    E *out, *gq, *gk, *gv;
    float *lse, *partial;
    // Of the rows, for the kernel of the keys: [heads, tokens] of each, stat_size apart: lse in units of log2, with the logarithm of what the row
    // of P sums to; -D; and with a bias lse as it is, and that logarithm.  (f16: both less 14, so that P comes times 2^14.)
    float* stats;
    int64_t stat_size;
    int32_t* lifts;            // f16, [heads, tokens / 32, 4]: the power of two that dS of 32 rows was held by, of each group of waves
    float *part_k, *part_v;    // with more than one part: [parts][tokens, kv_heads, dim] sums in f32
    int32_t head_parts, query_parts, partial_tiles;
    int* flag;
    uint16_t borders[ATTN_MAX_BUCKETS / 2];      // distance at which bucket exact_to + 1 + m begins
};

// ---- element types -----------------------------------------------------------------------------------------------------
template <class E> struct AttnType;
template <> struct AttnType<bf16_t> {
    using Frag = bf16x8_t;
    static constexpr int CHUNK = 8;       // elements in 16 bytes
    __device__ static f32x16_t mma(Frag a, Frag b, f32x16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    __device__ static Frag pack(f32x8_t x) { return __builtin_convertvector(x, bf16x8_t); }
    __device__ static u32x2_t pack4(f32x4_t x) { return __builtin_bit_cast(u32x2_t, __builtin_convertvector(x, bf16x4_t)); }
    __device__ static float get(bf16_t x) { return bf2f(x); }
    __device__ static bf16_t put(float x) { return f2bf(x); }
    __device__ static float get(Frag f, int e) { return (float)f[e]; }
};
template <> struct AttnType<f16_t> {
    using Frag = f16x8_t;
    static constexpr int CHUNK = 8;
    __device__ static f32x16_t mma(Frag a, Frag b, f32x16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    __device__ static Frag pack(f32x8_t x) { return __builtin_convertvector(x, f16x8_t); }
    __device__ static u32x2_t pack4(f32x4_t x) { return __builtin_bit_cast(u32x2_t, __builtin_convertvector(x, f16x4_t)); }
    __device__ static float get(f16_t x) { return h2f(x); }
    __device__ static f16_t put(float x) { return f2h(x); }
    __device__ static float get(Frag f, int e) { return (float)f[e]; }
};
template <> struct AttnType<float> {
    using Frag = f32x8_t;
    static constexpr int CHUNK = 4;
    // eight products of two terms each: term e of a lane's eight pairs the same index of both operands in either half
    __device__ static f32x16_t mma(Frag a, Frag b, f32x16_t c) {
#pragma unroll
        for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
    __device__ static Frag pack(f32x8_t x) { return x; }
    __device__ static float get(float x) { return x; }
    __device__ static float put(float x) { return x; }
    __device__ static float get(Frag f, int e) { return f[e]; }
};

__device__ inline float attn_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
// the value of the lane 32 further on (the other half of the same column)
__device__ inline float attn_other_half(float x) { return __shfl_xor(x, 32, WAVE); }

// ---- tiles in LDS ------------------------------------------------------------------------------------------------------
// ROWS rows of DP elements at a pitch of a power of two, in 16-byte pieces whose place within a row is XOR-ed with bits
// of the row: the 16 lanes that a 16-byte read serves together then meet all 64 banks once (32 rows, one piece each),
// and so do the transposed reads (4 rows, 4 neighbouring pieces each), for which rows 0..3 have to differ in the upper
// bits of the piece's place.
template <class E, int DP>
struct AttnTile {
    using T = AttnType<E>;
    using Frag = typename T::Frag;
    static constexpr int PITCH = (DP <= 32 ? 32 : DP <= 64 ? 64 : 128) * (int)sizeof(E);
    static constexpr int PIECES = PITCH / 16;                // of a row in LDS
    static constexpr int DATA = DP * (int)sizeof(E) / 16;    // of a row in memory (a multiple of 4)
    __device__ static int swizzle(int row) {
        if constexpr (PIECES >= 16) return ((row & 3) << 2) | ((row >> 2) & 3);
        else if constexpr (PIECES == 8) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
        else return (row >> 2) & 3;
    }
    __device__ static int at(int row, int piece) { return row * PITCH + ((piece ^ swizzle(row)) << 4); }
    // Where the fragments of a tile lie, for a lane.  A swizzle is made of bits of the row, so what is known when the
    // kernel is compiled (step, block, the row within 16) is an exclusive or and an offset to one register for each kind of
    // fragment; the tiles lie on multiples of their pitch.
    struct Lane {
        uint32_t rows, columns;
        __device__ explicit Lane(int lane) {
            const int r = lane & 31, half = lane >> 5;
            rows = at(r, sizeof(E) == 2 ? half : 2 * half);
            if constexpr (sizeof(E) == 2) {
                const int c = lane & 15;
                columns = at(4 * half + (c >> 2), 2 * ((lane >> 4) & 1) + ((c & 3) >> 1)) + (c & 1) * 8;
            } else {
                columns = at(4 * half, (lane & 31) >> 2) + (lane & 3) * 4;
            }
        }
    };
    template <class V>
    __device__ static V read(uint32_t from) { return *(__attribute__((address_space(3))) const V*)(uintptr_t)from; }
    // rows row0 + (lane % 32), elements 16 step + 8 half ..  (row0: a multiple of 32; base: the tile in LDS)
    __device__ static Frag rows(uint32_t base, const Lane& l, int row0, int step) {
        const uint32_t at = base + l.rows;
        if constexpr (sizeof(E) == 2) {
            return read<Frag>((at ^ (step << 5)) + row0 * PITCH);
        } else {
            const f32x4_t a = read<f32x4_t>((at ^ (step << 6)) + row0 * PITCH), b = read<f32x4_t>((at ^ (step << 6 | 16)) + row0 * PITCH);
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
    // column 32 block + (lane % 32), rows row0 + 4 half + (e % 4) + 8 (e / 4): the order in which a result holds its rows (row0: a
    // multiple of 16)
    __device__ static Frag columns(uint32_t base, const Lane& l, int row0, int block) {
        const uint32_t at = base + l.columns;
        if constexpr (sizeof(E) == 2) {
            // the hardware's transposed read: 16 lanes bring 4 rows x 16 columns, lane c gets column c
            const s16x4_t lo = read4((at ^ (block << 6)) + row0 * PITCH), hi = read4((at ^ (block << 6 ^ swizzle(8) << 4)) + (row0 + 8) * PITCH);
            return __builtin_bit_cast(Frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            Frag f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int r = (e & 3) + 8 * (e >> 2);
                f[e] = read<float>((at ^ (block << 7 ^ swizzle(r) << 4)) + (row0 + r) * PITCH);
            }
            return f;
        }
    }
    __device__ static s16x4_t read4(uint32_t from) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(uintptr_t)from); }
};
__device__ inline uint32_t attn_in_lds(const void* p) { return (uint32_t)(uintptr_t)p; }      // the low half of an address in LDS

// 16 bytes of a row from element d on, zeros beyond dim
template <class E>
__device__ inline u32x4_t attn_piece(const E* row, int d, int dim, int64_t elem, int vec) {
    constexpr int N = AttnType<E>::CHUNK;
    u32x4_t r = {0, 0, 0, 0};
    if (vec) {
        if (d < dim) r = *(const u32x4_t*)(row + d);
        return r;
    }
    E x[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
        x[e] = E{};
        if (d + e < dim) x[e] = row[(int64_t)(d + e) * elem];
    }
    __builtin_memcpy(&r, x, 16);
    return r;
}

// ROWS tokens of one operand, from memory to a tile in LDS.  Rows are whole 16-byte pieces in the usual case: they go
// straight to LDS (a wave's instruction fills 1 KB in a row; which piece of which row a lane fetches undoes the swizzle), with no
// register in between, and are waited for a tile later.  The compiler does not know of these loads, so that it does not wait for
// them before every read of LDS: attn_arrived() does, in front of the barrier that hands a tile over.  Anything else
// (other strides, heads that are not whole pieces) goes through registers, element by element.
// A token behind the last one that counts is replaced by that one: the mask hides what it brings.
template <int N>
__device__ inline void attn_wait() { asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory"); }

// the lane's number, found where it is asked for
__device__ inline int attn_lane() {
    int lane;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane));
    return lane;
}
// BYTES (4 or 16) of every lane, from base + off to 64 * BYTES of LDS in a row.  (m0, the place in LDS, is read as the load is
// issued; nothing else in these kernels uses it.)
template <int BYTES>
__device__ __forceinline__ void attn_load_lds(const void* base, uint32_t off, uint32_t to) {
    const uint64_t at = (uint64_t)(uintptr_t)base;
    const uint64_t from = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(at >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)at);
    const uint32_t place = (uint32_t)__builtin_amdgcn_readfirstlane((int)to);
    if constexpr (BYTES == 16) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" :: "s"(place), "v"(off), "s"(from) : "memory");
    else asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" :: "s"(place), "v"(off), "s"(from) : "memory");
}

// GROUP waves move the tiles of their own ring; `wave` is a wave's number among them.
template <class E, int DP, int ROWS, int GROUP>
struct AttnStage {
    using L = AttnTile<E, DP>;
    using Share = AttnShare<ROWS, L::PITCH, GROUP>;
    static constexpr int N = Share::N;                         // wave instructions of a wave for a tile
    // A wave's instructions bring rows that are STRIDE apart: where the swizzle is the same for them, one offset serves all, and
    // the rest is in the base.
    static constexpr int STRIDE = GROUP * 64 / L::PIECES;
    static constexpr bool ALIKE = STRIDE % 16 == 0;
    __device__ static int row_of(int u, int wave, int lane) { return Share::row_of(u, wave, lane); }
    __device__ static int piece_of(int u, int wave, int lane) { return (lane % L::PIECES) ^ L::swizzle(row_of(u, wave, lane)); }
    // bytes from the tile's first token to the lane's piece
    __device__ static uint32_t offset(const AttnView<E>& view, int u, int wave, int lane) {
        return ((uint32_t)row_of(u, wave, lane) * (uint32_t)view.token + piece_of(u, wave, lane) * L::T::CHUNK) * (uint32_t)sizeof(E);
    }
    // whether every lane brings a piece of every tile that lies within the walk: then a tile's loads are plain() ones.  (Rows of 96
    // elements have a pitch of 128: a lane that has no piece of the row must not reach for one.)
    __device__ static bool plainly(const AttnView<E>& view, int dim) { return view.vec && dim == DP && L::DATA == L::PIECES; }
    uint32_t kept;
    __device__ __forceinline__ AttnStage(const AttnView<E>& view, int wave, int lane) : kept(offset(view, 0, wave, lane)) {}
    __device__ __forceinline__ void plain(const AttnView<E>& view, const E* base, uint32_t tile, int wave) const {
        const int lane = attn_lane();
#pragma unroll
        for (int u = 0; u < N; ++u)
            attn_load_lds<16>(ALIKE ? base + u * STRIDE * view.token : base, ALIKE ? kept : offset(view, u, wave, lane), tile + Share::call_of(u, wave) * 1024);
    }
    // any tile that begins at a token before hi
    __device__ static __forceinline__ void load(const AttnView<E>& view, int head, int token0, int hi, int dim, char* tile, int wave, int lane) {
        const E* const base = view.p + (int64_t)head * view.head + (int64_t)token0 * view.token;
        if (view.vec) {
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const int row = row_of(u, wave, lane), piece = piece_of(u, wave, lane), in = token0 + row < hi ? row : hi - 1 - token0;
                const uint32_t from = (uint32_t)(in * (int)view.token + piece * L::T::CHUNK) * (uint32_t)sizeof(E);
                if (piece * L::T::CHUNK < dim) attn_load_lds<16>(base, from, attn_in_lds(tile) + Share::call_of(u, wave) * 1024);
            }
        } else {
#pragma nounroll
            for (int slot = wave * 64 + lane; slot < ROWS * L::PIECES; slot += GROUP * 64) {
                const int row = slot / L::PIECES, piece = (slot % L::PIECES) ^ L::swizzle(row), in = token0 + row < hi ? row : hi - 1 - token0;
                *(u32x4_t*)(tile + slot * 16) = attn_piece<E>(base + (int64_t)in * view.token, piece * L::T::CHUNK, dim, view.elem, 0);
            }
            attn_wait<0>();        // fewer loads than are counted for a tile: so none of those before stays on its way
        }
    }
};
// pieces that no load brings (dim below the pitch) have to be zeros: once, for all tiles that lie there later
__device__ inline void attn_clear(char* tiles, int bytes, int tid, int threads) {
    for (int at = tid * 16; at < bytes; at += threads * 16) *(u32x4_t*)(tiles + at) = u32x4_t{0, 0, 0, 0};
}

// Row fragments straight from memory, held for the whole loop; `sign` 1, -1 or 0 is multiplied in (exact).
template <class E, int DP>
__device__ inline void attn_own_rows(const AttnView<E>& view, int head, int token, bool there, int dim, int lane, float sign, typename AttnType<E>::Frag (&f)[DP / 16]) {
    using T = AttnType<E>;
    const E* row = view.p + (int64_t)head * view.head + (int64_t)token * view.token;
    const uint32_t flip = sizeof(E) == 2 ? 0x80008000u : 0x80000000u;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        u32x4_t part[sizeof(E) / 2];
#pragma unroll
        for (int c = 0; c < (int)sizeof(E) / 2; ++c) {
            part[c] = u32x4_t{0, 0, 0, 0};
            if (there && sign != 0.0f) part[c] = attn_piece<E>(row, 16 * s + 8 * (lane >> 5) + c * T::CHUNK, dim, view.elem, view.vec);
            if (sign < 0.0f) part[c] ^= flip;
        }
        __builtin_memcpy(&f[s], part, sizeof(f[s]));
    }
}

// ---- sequences -----------------------------------------------------------------------------------------------------------
// First token of the sequence of `row` and the first token behind it; false if no sequence holds the row.  Offsets that
// do not ascend give some bounds with first <= row < last <= tokens: never an access outside the tensors.
// CHECK: one wave of the first block looks the offsets over; the host reports what it finds with the next status.
template <bool CHECK, class E>
__device__ __forceinline__ bool attn_sequence(const AttnArgs<E>& a, int row, int lane, int& first, int& last) {
    const int32_t* const offsets = a.offsets;
    const int sequences = a.sequences, tokens = a.tokens;
    const bool looks = CHECK && blockIdx.x == 0 && threadIdx.x < WAVE;
    int lo = -1, hi = tokens;
    bool above = false;
    if (sequences < WAVE) {
        const int mine = lane <= sequences ? offsets[lane] : -1;
        if (looks) {
            const int next = __shfl_down(mine, 1, WAVE);
            if (lane <= sequences && (mine < 0 || mine > tokens || (lane < sequences && next < mine))) *a.flag = 1;
        }
        for (int e = 0; e <= sequences; ++e) {
            const int off = __builtin_amdgcn_readlane(mine, e);
            attn_take_offset(off, row, lo, hi, above);
        }
    } else {
        if (looks)
            for (int e = lane; e <= sequences; e += WAVE) {
                const int off = offsets[e];
                if (off < 0 || off > tokens || (e < sequences && offsets[e + 1] < off)) *a.flag = 1;
            }
        attn_search(offsets, sequences, row, lo, hi, above);
    }
    return attn_bounds(row, tokens, lo, hi, above, first, last);
}
// tile of rows and head of a block.  The blocks of a tile follow one another (the longest first); with a multiple of eight
// heads, neighbouring heads - which share their keys - are eight blocks apart: on one XCD, behind one L2.
__device__ inline void attn_place(int block, int tiles, int heads, bool last_first, int& tile, int& head) {
    const int t = block / heads, x = block - t * heads;
    tile = __builtin_amdgcn_readfirstlane(last_first ? tiles - 1 - t : t);
    head = __builtin_amdgcn_readfirstlane(heads % 8 == 0 ? (x % 8) * (heads / 8) + x / 8 : x);
}

// ---- the bias ------------------------------------------------------------------------------------------------------------
template <class E>
__device__ inline int attn_bucket(const AttnArgs<E>& a, int distance) {
    if (distance < a.exact_to) return distance;
    int b = a.exact_to;
    for (int m = 0; m < a.buckets - a.exact_to - 1; ++m) b += distance >= (int)a.borders[m];
    return b;
}
template <class E>
__device__ inline float attn_bias(const AttnArgs<E>& a, int head, int bucket) { return AttnType<E>::get(a.table[(int64_t)bucket * a.heads + head]); }
// by_distance[n], n = 0 .. max_distance: the bias of a head, the last for every distance from max_distance on
template <class E>
__device__ inline void attn_bias_by_distance(const AttnArgs<E>& a, int head, float* by_distance, int tid, int threads) {
    for (int n = tid; n <= a.max_distance; n += threads) by_distance[n] = attn_bias(a, head, attn_bucket(a, n));
}
// Every distance from max_distance on has one bias: a tile of such pairs starts its product there (in units of the product),
// and costs nothing.  A bias is any finite number, the type's lowest value among them, and rows may hold nothing else: there q . k is
// lost beside it, and what decides is that equal scores stay equal.  So a large one goes the way of a near tile, where scores
// are formed as they are defined, and the maximum and lse with them: only their differences are brought to units of log2.
// how many of n tiles, a step apart, lie at `room` or before it, the first lying at 0
__device__ __forceinline__ int attn_tiles_beyond(int room, int step, int n) {
    const int fit = room < 0 ? 0 : room / step + 1;
    return fit < n ? fit : n;
}
struct AttnFar {
    float start;
    bool apart;
    __device__ __forceinline__ AttnFar(float bias, float scale)
        : start(bias / scale), apart(!(__builtin_fabsf(bias) < 1024.0f && __builtin_fabsf(bias) < 1e30f * scale) && bias != -INFINITY) {}
};
// The scores that a lane holds at distances d0 - (r % 4) - 8 (r / 4), times STEP (1: rows are keys, -1: queries)
template <int STEP>
__device__ inline void attn_add_bias(f32x16_t& s, float scale, const float* by_distance, int d0, int max_distance) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        int n = d0 - STEP * ((r & 3) + 8 * (r >> 2));
        n = n < 0 ? 0 : n > max_distance ? max_distance : n;
        s[r] = __builtin_fmaf(s[r], scale, by_distance[n]);
    }
}
__device__ inline f32x16_t attn_start(float x) {
    f32x16_t s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = x;
    return s;
}

// ---- what a mask hides -----------------------------------------------------------------------------------------------------
// The matrix cores multiply a weight of zero by whatever the other operand holds: a NaN or an infinity in a row that the mask hides
// from a column (a later token, another sequence) would become a NaN there.  So the tiles that a mask touches - a few at either end
// of a block's walk, in a loop of their own - are looked over, and one that holds such a value is added term by term:
// sums[d] += weight * tile[row][d] for the rows that `sees` lets through.
template <class E>
__device__ inline bool attn_finite(u32x4_t x) {
    bool fine = true;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (sizeof(E) == 4) {
            fine &= (x[e] & 0x7F800000u) != 0x7F800000u;
        } else {
            const uint32_t exponent = std::is_same<E, bf16_t>::value ? 0x7F80u : 0x7C00u;
            fine &= (x[e] & exponent) != exponent && (x[e] >> 16 & exponent) != exponent;
        }
    }
    return fine;
}
// by the GROUP waves of a ring (tid among their threads), the tile being there: whether it holds such a value.  All waves of the block
// come along.
template <class E, int GROUP>
__device__ __forceinline__ bool attn_look_over(const char* tile, int bytes, int* said, int tid, int lane) {
    bool fine = true;
    for (int at = tid * 16; at < bytes; at += GROUP * 64 * 16) fine &= attn_finite<E>(*(const u32x4_t*)(tile + at));
    const bool any = __any(!fine);
    if (lane == 0) said[tid >> 6] = any;
    __syncthreads();
    int bad = 0;
#pragma unroll
    for (int w = 0; w < GROUP; ++w) bad |= said[w];
    return __builtin_amdgcn_readfirstlane(bad) != 0;
}
template <class E, int DP, int TILES, class Sees>
__device__ __forceinline__ void attn_add_terms(const char* tile, const f32x16_t (&weight)[TILES], f32x16_t (&sums)[DP / 32], int lane, Sees sees) {
    using L = AttnTile<E, DP>;
    const int half = lane >> 5;
#pragma nounroll
    for (int row = 0; row < 32 * TILES; ++row) {
        const int at = (row & 3) + 4 * ((row >> 3) & 3) + 16 * (row >> 5);      // where the lane's half of rows keeps it
        float mine = 0.0f;
#pragma unroll
        for (int r = 0; r < 16 * TILES; ++r) mine = r == at ? weight[r >> 4][r & 15] : mine;
        const float w = __shfl(mine, (lane & 31) | (((row >> 2) & 1) << 5), WAVE);
        const bool seen = sees(row);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c0 = 32 * d + 8 * g + 4 * half;
                E x[4];
                __builtin_memcpy(x, tile + L::at(row, c0 * (int)sizeof(E) / 16) + c0 * (int)sizeof(E) % 16, sizeof(x));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float y = __builtin_fmaf(w, AttnType<E>::get(x[e]), sums[d][4 * g + e]);
                    sums[d][4 * g + e] = seen ? y : sums[d][4 * g + e];
                }
                __builtin_amdgcn_sched_barrier(0);       // a few registers at a time
            }
    }
}
// sums[d] += weight^T tile, the summed index in the rows of both
template <class E, int DP>
__device__ __forceinline__ void attn_add_product(uint32_t tile, const typename AttnTile<E, DP>::Lane& l, int row0, const f32x16_t& weight, f32x16_t (&sums)[DP / 32]) {
    using T = AttnType<E>;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        f32x8_t p;
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = weight[8 * h + e];
        const typename T::Frag pf = T::pack(p);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) sums[d] = T::mma(AttnTile<E, DP>::columns(tile, l, row0 + 16 * h, d), pf, sums[d]);
    }
}

// the tile at the ring's place has come, and the one before it is done with by all waves
template <int PER>
__device__ __forceinline__ void attn_arrived(const AttnRing& ring) {
    static_assert(3 * PER < 64, "the counter has six bits");
    const int later = ring.later();
    if (later >= 3) attn_wait<3 * PER>();
    else if (later == 2) attn_wait<2 * PER>();
    else if (later == 1) attn_wait<PER>();
    else attn_wait<0>();
    __syncthreads();
}
// Kinds of tiles, each in a loop of its own.  (Clean ones that lie beyond max_distance for every row of the block, with one bias for all
// pairs, are a kind where that pays: in the kernel of the keys up to 64 elements a head, 280 -> 262 us.  The others lose by it.)
enum { ATTN_FAR, ATTN_CLEAN, ATTN_MASKED };
template <int KIND> using AttnKind = std::integral_constant<int, KIND>;
template <int PER, class Rounds, class Fetch, class Step>
__device__ __forceinline__ void attn_run_rounds(const Rounds& rounds, AttnRing& ring, Fetch&& fetch, Step&& step) {
    auto turn = [&](auto kind, int round) __attribute__((always_inline)) {
        attn_arrived<PER>(ring);
        ring.refill(fetch);
        step(kind, round, ring.at);
        ring.done();
    };
    int round = 0;
    for (; round < rounds.clean; ++round) turn(AttnKind<ATTN_CLEAN>{}, round);
    for (; round < rounds.total; ++round) turn(AttnKind<ATTN_MASKED>{}, round);
}

// the span of a wave's 32 rows: a lane's row sees [from, upto)
__device__ __forceinline__ AttnSpan attn_span(bool there, int from, int upto) {
    const uint32_t rows = (uint32_t)__ballot(there);           // (the halves of a wave say the same)
    if (rows == 0) return AttnSpan();
    const int a = __builtin_ctz(rows), b = 31 - __builtin_clz(rows);
    return AttnSpan(__builtin_amdgcn_readlane(from, a), __builtin_amdgcn_readlane(upto, a), __builtin_amdgcn_readlane(from, b), __builtin_amdgcn_readlane(upto, b));
}
// of the rows of WAVES waves
template <int WAVES>
__device__ __forceinline__ AttnSpan attn_span_of_block(const AttnSpan& own, int* shared, int wave, int lane) {
    if (lane == 0) own.put(shared + 4 * wave);
    __syncthreads();
    AttnSpan all;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) all.join(shared + 4 * w);
    all.close();
    all.lo = __builtin_amdgcn_readfirstlane(all.lo);
    all.hi = __builtin_amdgcn_readfirstlane(all.hi);
    all.inner = __builtin_amdgcn_readfirstlane(all.inner);
    all.top = __builtin_amdgcn_readfirstlane(all.top);
    return all;
}

// f16 has no room for dS as it comes: a loss that is scaled up takes it beyond 65504, a mean over many tokens below 2^-24, long before the
// gradients leave the type.  A wave holds it, and the sum it goes into, times 2^-e: the first values that are not zero come to lie
// around 2^10, and e grows when some reach 2^15.  What gets lost in subnormals is 2^-35 of the largest.  The kernel of the queries finds e as
// it goes and leaves it for the kernel of the keys, which takes the largest of the rows that it walks over.  (P, which is never above one,
// is held times 2^14 there.)  8192 tokens, 16 heads: the kernel of the queries 130 -> 139 us at 64 elements, 205 -> 209 at 128, that of the
// keys 233 -> 247 and 466 -> 470; with e found in both, 272 and 560.
template <class E> constexpr bool attn_lifted() { return std::is_same<E, f16_t>::value; }
template <class E> constexpr int attn_p_up() { return attn_lifted<E>() ? 14 : 0; }
constexpr int ATTN_NO_LIFT = -1000;         // nothing but zeros
struct AttnLift {
    float limit = 0.0f;
    int e = 0;
    template <int DB>
    __device__ __forceinline__ void hold(f32x16_t& s, f32x16_t (&sums)[DB], float& other) {
        float top = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, __builtin_fabsf(s[r]));
        if (__any(top > limit)) {
            top = 0.0f;                         // (an infinite value stays one, and says nothing about the other rows)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = __builtin_fabsf(s[r]) < INFINITY ? fmaxf(top, __builtin_fabsf(s[r])) : top;
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, WAVE));
            if (!(top > limit)) return;
            int up = 11 - __builtin_amdgcn_frexp_expf(top);
            up = up < e - 100 ? e - 100 : up > e + 80 ? e + 80 : up;      // (dS is below 2^40: nothing overflows in f32)
            up = __builtin_amdgcn_readfirstlane(up);
            const float by = power(up);
            s *= attn_start(by);
#pragma unroll
            for (int d = 0; d < DB; ++d) sums[d] *= attn_start(by);
            other *= by;
            e -= up;
            limit = 32768.0f;
        }
    }
    __device__ static __forceinline__ float power(int n) { return __builtin_ldexpf(1.0f, n); }
};

// the largest power of the rows of `heads` heads that a block walks over, found by its waves together
template <class E>
__device__ __forceinline__ int attn_lift_of_rows(const AttnArgs<E>& a, int head0, int heads, const AttnSpan& all, int* shared, int tid, int lane, int wave) {
    const int from = all.lo / 32, n = all.hi > all.lo ? (all.hi - 1) / 32 + 1 - from : 0, chunks = (a.tokens + 31) / 32;
    int e = ATTN_NO_LIFT;
    for (int x = tid; x < n * heads; x += ATTN_THREADS) {
        const int h = x / n;
        const int32_t* const four = a.lifts + ((int64_t)(head0 + h) * chunks + from + x - h * n) * 4;
#pragma unroll
        for (int g = 0; g < 4; ++g) e = four[g] > e ? four[g] : e;
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        const int other = __shfl_xor(e, d, WAVE);
        e = other > e ? other : e;
    }
    __syncthreads();
    if (lane == 0) shared[wave] = e;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < ATTN_WAVES; ++w) e = shared[w] > e ? shared[w] : e;
    e = e < -80 ? 0 : e > 100 ? 100 : e;       // (nothing found, or offsets that do not ascend)
    return __builtin_amdgcn_readfirstlane(e);
}

// Sums of another group of waves for the same rows, through LDS: `count` registers of a wave, four at a time.
template <int DB>
__device__ inline void attn_leave(float* to, const f32x16_t (&sums)[DB], float x, float y, int lane) {
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) *(f32x4_t*)(to + ((4 * d + g) * 64 + lane) * 4) = f32x4_t{sums[d][4 * g], sums[d][4 * g + 1], sums[d][4 * g + 2], sums[d][4 * g + 3]};
    to[DB * 1024 + lane] = x;
    to[DB * 1024 + 64 + lane] = y;
}
template <int DB>
__device__ inline void attn_take(const float* from, f32x16_t (&sums)[DB], float by, float from_by, int lane) {
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4_t x = *(const f32x4_t*)(from + ((4 * d + g) * 64 + lane) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) sums[d][4 * g + e] = __builtin_fmaf(x[e], from_by, sums[d][4 * g + e] * by);
        }
}
template <int DB> constexpr int attn_left() { return DB * 1024 + 128; }       // floats of a wave

// rows of a result (index in the columns of the fragments), four neighbouring elements at a time where they lie on their boundaries
template <class E, int DP>
__device__ inline void attn_write_row(E* out, const f32x16_t (&sums)[DP / 32], float by, int dim, int half, bool whole) {
    using T = AttnType<E>;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int at = 32 * d + 8 * g + 4 * half;
            E x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = T::put(sums[d][4 * g + e] * by);
            if (whole) {
                if (at < dim) __builtin_memcpy(__builtin_assume_aligned(out + at, 4 * sizeof(E)), x, sizeof(x));
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (at + e < dim) out[at + e] = x[e];
            }
        }
}
template <class E>
__device__ inline bool attn_whole(const E* out, int dim) { return dim % 4 == 0 && (uintptr_t)out % (4 * sizeof(E)) == 0; }

__device__ inline float attn_sign(float scale) { return scale > 0.0f ? 1.0f : scale < 0.0f ? -1.0f : scale == 0.0f ? 0.0f : 1.0f; }

// ---- forward -------------------------------------------------------------------------------------------------------------
// One pass over the keys with a running maximum and sum.  A matrix instruction takes 1 KB of keys or values from LDS, which keeps LDS as
// busy as the matrix cores: bf16, 8192 tokens (5000, 2500, 692), 32 heads of 128 sharing 8: 300 us = 868 TFLOP/s, where a
// large product reaches 1202.
// KG groups of waves share a walk; four of them own 64 rows (two waves each), not 128.  Keys of a tile: 64 KB of LDS for two tiles of keys
// and values of a group, 32 KB where four groups have rings.
template <int KG> constexpr int attn_row_waves() { return KG == 4 ? 2 : ATTN_ROWS / 32; }
template <class E, int DP, int KG> constexpr int attn_keys() { return sizeof(E) == 4 || (KG == 4 && DP > 64) ? 32 : 64; }
template <class E, int DP>
constexpr size_t attn_tile_bytes(int rows) { return (size_t)rows * AttnTile<E, DP>::PITCH; }
// the running maximum may be this much (a factor of 2^8) behind before the sums are rescaled
constexpr float ATTN_BEHIND = 8.0f;

template <class E, int DP, bool BIAS, int KG>
__global__ __launch_bounds__(64 * attn_row_waves<KG>() * KG, sizeof(E) == 4 && DP > 64 ? 1 : 2) void attn_forward_kernel(const AttnArgs<E> a, int tiles, int stages) {
    using T = AttnType<E>;
    using L = AttnTile<E, DP>;
    constexpr int RG = attn_row_waves<KG>(), BN = attn_keys<E, DP, KG>(), JB = BN / 32, DB = DP / 32, KS = DP / 16, BYTES = BN * L::PITCH;
    extern __shared__ __attribute__((aligned(512))) char lds[];
    __shared__ int span[4 * RG * KG];
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, group = __builtin_amdgcn_readfirstlane(tid / (64 * RG)), wave = __builtin_amdgcn_readfirstlane(tid / 64 % RG);
    char* const mine = lds + group * stages * 2 * BYTES;         // the group's ring
    const typename L::Lane at(lane);
    int* const said = span + group * RG;
    float* const by_distance = (float*)(lds + KG * stages * 2 * BYTES);
    int tile, head;
    attn_place(blockIdx.x, tiles, a.heads, true, tile, head);
    const int kv = head / a.group;
    const int row0 = tile * (32 * RG) + wave * 32, row = row0 + (lane & 31);
    int first, last;
    const bool there = attn_sequence<true>(a, row, lane, first, last);
    const AttnSpan own = attn_span(there, first, row + 1), all = attn_span_of_block<RG>(own, span, wave, lane);      // keys
    if (all.hi <= all.lo) return;                   // no row of the block is in a sequence
    const AttnStage<E, DP, BN, RG> ks(a.k, wave, lane), vs(a.v, wave, lane);
    const AttnWalk<BN> walk(all.lo, all.hi, all.inner, all.top);
    const AttnRounds<AttnWalk<BN>, KG> rounds(walk, group);
    if (a.dim * (int)sizeof(E) < L::PITCH) {
        attn_clear(lds, KG * stages * 2 * BYTES, tid, 64 * RG * KG);
        __syncthreads();
    }
    AttnRing ring(stages);
    // the next round's tiles: while they are clean ones, a group's follow one another at a fixed distance
    const int plain = ks.plainly(a.k, a.dim) && vs.plainly(a.v, a.dim) ? walk.nclean / KG : 0;
    const int64_t to_next_k = (int64_t)(KG * BN) * a.k.token, to_next_v = (int64_t)(KG * BN) * a.v.token;
    const E *next_k = a.k.p + (int64_t)kv * a.k.head + (int64_t)walk.at(group) * a.k.token, *next_v = a.v.p + (int64_t)kv * a.v.head + (int64_t)walk.at(group) * a.v.token;
    int next = 0;
    auto fetch = [&](int place) __attribute__((always_inline)) {
        char* const to = mine + place * 2 * BYTES;
        if (next < plain) {
            ks.plain(a.k, next_k, attn_in_lds(to), wave);
            vs.plain(a.v, next_v, attn_in_lds(to) + BYTES, wave);
            next_k += to_next_k;
            next_v += to_next_v;
        } else {
            const int j0 = walk.at(rounds.nearest(next));
            ks.load(a.k, kv, j0, all.hi, a.dim, to, wave, lane);
            vs.load(a.v, kv, j0, all.hi, a.dim, to + BYTES, wave, lane);
        }
        ++next;
    };
    ring.begin(rounds.total, fetch);
    typename T::Frag q[KS];
    attn_own_rows<E, DP>(a.q, head, there ? row : 0, there, a.dim, lane, attn_sign(a.scale), q);
    if (BIAS) attn_bias_by_distance(a, head, by_distance, tid, 64 * RG * KG);
    const AttnFar far(BIAS ? attn_bias(a, head, a.buckets - 1) : 0.0f, a.scale_abs);

    const int lower = there ? first : -1;           // key j is seen if (unsigned)(j - lower) <= reach
    const uint32_t reach = there ? (uint32_t)(row - first) : 0;
    const float c = a.scale_log2;
    f32x16_t acc[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[d] = f32x16_t{};
    constexpr float UNIT = BIAS ? ATTN_LOG2E : 1.0f;          // of the maximum: as scores are with a bias, else of log2
    float m = -INFINITY, l = 0.0f;
    auto step = [&](auto kind_, int round, int place) __attribute__((always_inline)) {
        constexpr bool MASKED = decltype(kind_)::value == ATTN_MASKED;
        const char* const kt = mine + place * 2 * BYTES;
        const char* const vt = kt + BYTES;
        const int n = rounds.tile(round), j0 = walk.at(n);
        const bool idle = KG > 1 && n >= (MASKED ? walk.total : walk.nclean);
        if (!MASKED && idle) return;
        bool terms = false;
        if constexpr (MASKED) {
            terms = attn_look_over<E, RG>(vt, BYTES, said, tid % (64 * RG), lane);
            if (idle || j0 >= own.hi || j0 + BN <= own.lo) return;
        }
        f32x16_t s[JB];
        const bool near = BIAS && (far.apart || row0 - (j0 + BN - 1) < a.max_distance);
#pragma unroll
        for (int b = 0; b < JB; ++b) {
            s[b] = attn_start(BIAS && !near ? far.start : 0.0f);
#pragma unroll
            for (int k = 0; k < KS; ++k) s[b] = T::mma(L::rows(attn_in_lds(kt), at, 32 * b, k), q[k], s[b]);
        }
        const int j = j0 + 4 * half;                // key of row 0 of the lane's results
        if (BIAS && near) {
#pragma unroll
            for (int b = 0; b < JB; ++b) attn_add_bias<1>(s[b], a.scale_abs, by_distance, row - j - 32 * b, a.max_distance);
        }
        if constexpr (MASKED) {
#pragma unroll
            for (int b = 0; b < JB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if ((uint32_t)(j + 32 * b + (r & 3) + 8 * (r >> 2) - lower) > reach) s[b][r] = -INFINITY;
        }
        float best = s[0][0];
#pragma unroll
        for (int b = 0; b < JB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) best = fmaxf(best, s[b][r]);
        best = fmaxf(best, attn_other_half(best));
        best *= BIAS ? near ? 1.0f : a.scale_abs : c;
        if (__any(best > m + ATTN_BEHIND / UNIT)) {
            const float next = fmaxf(m, best), fix = next == -INFINITY ? 1.0f : attn_exp2((m - next) * UNIT);
            l *= fix;
#pragma unroll
            for (int d = 0; d < DB; ++d) acc[d] *= fix;
            m = next;
        }
        const float base = m == -INFINITY ? 0.0f : m;
        if (BIAS && near) {
#pragma unroll
            for (int b = 0; b < JB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[b][r] = (s[b][r] - base) * ATTN_LOG2E;
        } else {
            const float base2 = base * UNIT;
#pragma unroll
            for (int b = 0; b < JB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[b][r] = __builtin_fmaf(s[b][r], c, -base2);
        }
#pragma unroll
        for (int b = 0; b < JB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[b][r] = attn_exp2(s[b][r]);
                l += s[b][r];
            }
        if (MASKED && terms) {
            attn_add_terms<E, DP, JB>(vt, s, acc, lane, [&](int r) __attribute__((always_inline)) { return (uint32_t)(j0 + r - lower) <= reach; });
        } else {
#pragma unroll
            for (int b = 0; b < JB; ++b) attn_add_product<E, DP>(attn_in_lds(vt), at, 32 * b, s[b], acc);
        }
    };
    attn_run_rounds<2 * AttnStage<E, DP, BN, RG>::N>(rounds, ring, fetch, step);
    if constexpr (KG > 1) {
        __syncthreads();                            // the rings are not needed any more
        float* const left = (float*)lds;
        if (group > 0) attn_leave<DB>(left + ((group - 1) * RG + wave) * attn_left<DB>(), acc, m, l, lane);
        __syncthreads();
        if (group > 0) return;
        for (int g = 1; g < KG; ++g) {
            const float* const from = left + ((g - 1) * RG + wave) * attn_left<DB>();
            const float m2 = from[DB * 1024 + lane], l2 = from[DB * 1024 + 64 + lane], next = fmaxf(m, m2);
            const float by = next == -INFINITY ? 1.0f : attn_exp2((m - next) * UNIT), by2 = next == -INFINITY ? 1.0f : attn_exp2((m2 - next) * UNIT);
            attn_take<DB>(from, acc, by, by2, lane);
            l = __builtin_fmaf(l2, by2, l * by);
            m = next;
        }
    }
    l += attn_other_half(l);
    if (!there) return;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;       // nothing but -inf: an output of zeros
    const float log_l = __builtin_amdgcn_logf(l);
    if (half == 0) a.lse[(int64_t)head * a.tokens + row] = l == 0.0f ? -INFINITY : BIAS ? __builtin_fmaf(log_l, ATTN_LN2, m) : (m + log_l) * ATTN_LN2;
    attn_write_row<E, DP>(a.out + ((int64_t)row * a.heads + head) * a.dim, acc, inv, a.dim, half, attn_whole(a.out, a.dim));
}

// ---- backward: gradients of the queries ------------------------------------------------------------------------------------
// A block owns 128 queries like the forward kernel.  Writes dq (if wanted) and, for the kernel of the keys, lse and D_i: with a
// bias the one that makes the row of dS sum to zero (formed from P and dP themselves; the rounding of o in do . o
// would otherwise enter every pair of the far bucket with the same sign).  bf16, 8192 tokens (4096, 3000, 1096), 16 heads of 128: 196-217
// us = 760-846 TFLOP/s, 16 heads of 64: 110 us.
// The sum, the rows of q and those of do take 128 registers at 128 elements a head.  With 64 keys to a tile the rest does not suffice (a
// register more than there are is read from memory, behind every tile on its way): 8192 tokens, 16 heads with a bias 313 us, with 32
// keys 212.  (With a bias five registers are read back even so, for lse as it is: 214 us.)
//
// With a bias, scores and lse may be so large that lse has lost the logarithm of the sum to its rounding (masks by large negative numbers:
// the row of P would sum to the number of its keys).  Beyond ATTN_ROUGH - 2^8 2^-24 = 2^-16 - a wave forms that sum first, keys straight
// from memory: seldom, and slowly.
constexpr float ATTN_ROUGH = 256.0f;
template <class E, int DP>
__device__ inline float attn_row_sum(const AttnArgs<E>& a, int head, int kv, int row, int lane, const AttnSpan& own, int lower, uint32_t reach, float lse,
                                     const typename AttnType<E>::Frag (&q)[DP / 16]) {
    float z = 0.0f;
#pragma nounroll
    for (int j0 = own.lo; j0 < own.hi; j0 += 32) {
        const int j = j0 + (lane & 31) < own.hi ? j0 + (lane & 31) : j0;
        const E* const from = a.k.p + (int64_t)kv * a.k.head + (int64_t)j * a.k.token;
        f32x16_t s = {};
#pragma unroll
        for (int x = 0; x < DP / 16; ++x) {
            u32x4_t part[sizeof(E) / 2];
            for (int c = 0; c < (int)sizeof(E) / 2; ++c) part[c] = attn_piece<E>(from, 16 * x + 8 * (lane >> 5) + c * AttnType<E>::CHUNK, a.dim, a.k.elem, a.k.vec);
            s = AttnType<E>::mma(__builtin_bit_cast(typename AttnType<E>::Frag, part), q[x], s);
            __builtin_amdgcn_sched_barrier(0);       // a few registers at a time
        }
        float mine[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) mine[r] = s[r];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int key = j0 + 4 * (lane >> 5) + (r & 3) + 8 * (r >> 2);
            if ((uint32_t)(key - lower) <= reach) z += attn_exp2((__builtin_fmaf(mine[r], a.scale_abs, attn_bias(a, head, attn_bucket(a, row - key))) - lse) * ATTN_LOG2E);
        }
    }
    z += attn_other_half(z);
    return z > 0.0f ? z : 1.0f;      // (nothing in view, or NaN)
}
template <class E, int DP, int KG> constexpr int attn_grad_keys() { return sizeof(E) == 2 && DP > 96 ? 32 : attn_keys<E, DP, KG>(); }
template <class E, int DP, bool BIAS, int KG>
__global__ __launch_bounds__(64 * attn_row_waves<KG>() * KG, sizeof(E) == 4 && DP > 64 ? 1 : 2) void attn_grad_query_kernel(const AttnArgs<E> a, int tiles, int stages) {
    using T = AttnType<E>;
    using L = AttnTile<E, DP>;
    constexpr int RG = attn_row_waves<KG>(), BN = attn_grad_keys<E, DP, KG>(), JB = BN / 32, DB = DP / 32, KS = DP / 16, BYTES = BN * L::PITCH;
    extern __shared__ __attribute__((aligned(512))) char lds[];
    __shared__ int span[4 * RG * KG];
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, group = __builtin_amdgcn_readfirstlane(tid / (64 * RG)), wave = __builtin_amdgcn_readfirstlane(tid / 64 % RG);
    char* const mine = lds + group * stages * 2 * BYTES;         // the group's ring
    const typename L::Lane at(lane);
    int* const said = span + group * RG;
    float* const by_distance = (float*)(lds + KG * stages * 2 * BYTES);
    int tile, head;
    attn_place(blockIdx.x, tiles, a.heads, true, tile, head);
    const int kv = head / a.group;
    const int row0 = tile * (32 * RG) + wave * 32, row = row0 + (lane & 31);
    int first, last;
    const bool there = attn_sequence<true>(a, row, lane, first, last);
    const AttnSpan own = attn_span(there, first, row + 1), all = attn_span_of_block<RG>(own, span, wave, lane);      // keys
    if (all.hi <= all.lo) return;
    const AttnStage<E, DP, BN, RG> ks(a.k, wave, lane), vs(a.v, wave, lane);
    const AttnWalk<BN> walk(all.lo, all.hi, all.inner, all.top);
    const AttnRounds<AttnWalk<BN>, KG> rounds(walk, group);
    if (a.dim * (int)sizeof(E) < L::PITCH) {
        attn_clear(lds, KG * stages * 2 * BYTES, tid, 64 * RG * KG);
        __syncthreads();
    }
    AttnRing ring(stages);
    // the next round's tiles: while they are clean ones, a group's follow one another at a fixed distance
    const int plain = ks.plainly(a.k, a.dim) && vs.plainly(a.v, a.dim) ? walk.nclean / KG : 0;
    const int64_t to_next_k = (int64_t)(KG * BN) * a.k.token, to_next_v = (int64_t)(KG * BN) * a.v.token;
    const E *next_k = a.k.p + (int64_t)kv * a.k.head + (int64_t)walk.at(group) * a.k.token, *next_v = a.v.p + (int64_t)kv * a.v.head + (int64_t)walk.at(group) * a.v.token;
    int next = 0;
    auto fetch = [&](int place) __attribute__((always_inline)) {
        char* const to = mine + place * 2 * BYTES;
        if (next < plain) {
            ks.plain(a.k, next_k, attn_in_lds(to), wave);
            vs.plain(a.v, next_v, attn_in_lds(to) + BYTES, wave);
            next_k += to_next_k;
            next_v += to_next_v;
        } else {
            const int j0 = walk.at(rounds.nearest(next));
            ks.load(a.k, kv, j0, all.hi, a.dim, to, wave, lane);
            vs.load(a.v, kv, j0, all.hi, a.dim, to + BYTES, wave, lane);
        }
        ++next;
    };
    const bool walks = a.gq || BIAS || (attn_lifted<E>() && a.gk);       // else only D_i is wanted, if that
    if (walks) ring.begin(rounds.total, fetch);
    typename T::Frag q[KS], go[KS];
    attn_own_rows<E, DP>(a.go, head, there ? row : 0, there, a.dim, lane, 1.0f, go);
    float delta = 0.0f, lse = INFINITY;
    {
        attn_own_rows<E, DP>(a.o, head, there ? row : 0, there, a.dim, lane, 1.0f, q);
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) delta = __builtin_fmaf(T::get(go[k], e), T::get(q[k], e), delta);
        delta += attn_other_half(delta);
    }
    if (there) {
        lse = a.lse[(int64_t)head * a.tokens + row];
        if (lse == -INFINITY) lse = INFINITY;                    // a row of nothing but -inf: P is zero
    }
    float* const stat = a.stats + (int64_t)head * a.tokens + row;
    if (!walks) {
        if (there && half == 0 && group == 0) { stat[0] = lse * ATTN_LOG2E - attn_p_up<E>(); stat[a.stat_size] = -delta; }
        return;
    }
    attn_own_rows<E, DP>(a.q, head, there ? row : 0, there, a.dim, lane, attn_sign(a.scale), q);
    if (BIAS) attn_bias_by_distance(a, head, by_distance, tid, 64 * RG * KG);
    const AttnFar far(BIAS ? attn_bias(a, head, a.buckets - 1) : 0.0f, a.scale_abs);
    const int lower = there ? first : -1;
    const uint32_t reach = there ? (uint32_t)(row - first) : 0;
    const float c = a.scale_log2;
    if constexpr (BIAS) {                 // (kept in memory over the walk, where registers are scarce; both halves and all groups write the same)
        float z = 1.0f;
        const bool rough = __builtin_fabsf(lse) > ATTN_ROUGH && lse != INFINITY;
        if (__any(rough)) {
            const float sum = attn_row_sum<E, DP>(a, head, kv, row, lane, own, lower, reach, lse, q);
            z = rough ? sum : 1.0f;             // (the other rows are as they would be without these)
        }
        if (there) {
            stat[2 * a.stat_size] = lse;
            stat[3 * a.stat_size] = __builtin_amdgcn_logf(z) - attn_p_up<E>();
        }
    }
    f32x16_t acc[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[d] = f32x16_t{};
    float rest = 0.0f;
    AttnLift lift;
    auto step = [&](auto kind_, int round, int place) __attribute__((always_inline)) {
        constexpr bool MASKED = decltype(kind_)::value == ATTN_MASKED;
        const char* const kt = mine + place * 2 * BYTES;
        const char* const vt = kt + BYTES;
        const int n = rounds.tile(round), j0 = walk.at(n);
        const bool idle = KG > 1 && n >= (MASKED ? walk.total : walk.nclean);
        if (!MASKED && idle) return;
        bool terms = false;
        if constexpr (MASKED) {
            terms = attn_look_over<E, RG>(kt, BYTES, said, tid % (64 * RG), lane);
            if (idle || j0 >= own.hi || j0 + BN <= own.lo) return;
        }
        const bool near = BIAS && (far.apart || row0 - (j0 + BN - 1) < a.max_distance);
#pragma unroll
        for (int b = 0; b < JB; ++b) {
            f32x16_t s = attn_start(BIAS && !near ? far.start : 0.0f), dp = f32x16_t{};
#pragma unroll
            for (int k = 0; k < KS; ++k) s = T::mma(L::rows(attn_in_lds(kt), at, 32 * b, k), q[k], s);
#pragma unroll
            for (int k = 0; k < KS; ++k) dp = T::mma(L::rows(attn_in_lds(vt), at, 32 * b, k), go[k], dp);
            const int j = j0 + 32 * b + 4 * half;
            if (BIAS && near) {
                attn_add_bias<1>(s, a.scale_abs, by_distance, row - j, a.max_distance);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = attn_lifted<E>() ? __builtin_fmaf(s[r] - lse, ATTN_LOG2E, -(float)lift.e) : (s[r] - lse) * ATTN_LOG2E;
            } else {
                const float lse2 = attn_lifted<E>() ? __builtin_fmaf(lse, ATTN_LOG2E, (float)lift.e) : lse * ATTN_LOG2E;
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], c, -lse2);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[r] = attn_exp2(s[r]);
                s[r] *= dp[r] - delta;
                if (MASKED && (uint32_t)(j + (r & 3) + 8 * (r >> 2) - lower) > reach) s[r] = 0.0f;
                if (BIAS && !attn_lifted<E>()) rest += s[r];
            }
            if constexpr (attn_lifted<E>()) {
                lift.hold(s, acc, rest);
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (BIAS) rest += s[r];
            }
            if (MASKED && terms) {
                const f32x16_t w[1] = {s};
                attn_add_terms<E, DP, 1>(kt + 32 * b * L::PITCH, w, acc, lane, [&](int r) __attribute__((always_inline)) { return (uint32_t)(j0 + 32 * b + r - lower) <= reach; });
            } else {
                attn_add_product<E, DP>(attn_in_lds(kt), at, 32 * b, s, acc);
            }
        }
    };
    attn_run_rounds<2 * AttnStage<E, DP, BN, RG>::N>(rounds, ring, fetch, step);
    if constexpr (attn_lifted<E>()) {
        if (lane == 0 && row0 < a.tokens)
            for (int slot = group; slot < 4; slot += KG) a.lifts[((int64_t)head * ((a.tokens + 31) / 32) + row0 / 32) * 4 + slot] = lift.limit == 0.0f ? ATTN_NO_LIFT : lift.e;
        const float by = AttnLift::power(lift.e);
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[d] *= attn_start(by);
        rest *= by;
    }
    if constexpr (KG > 1) {
        __syncthreads();
        float* const left = (float*)lds;
        if (group > 0) attn_leave<DB>(left + ((group - 1) * RG + wave) * attn_left<DB>(), acc, rest, 0.0f, lane);
        __syncthreads();
        if (group > 0) return;
        for (int g = 1; g < KG; ++g) {
            const float* const from = left + ((g - 1) * RG + wave) * attn_left<DB>();
            attn_take<DB>(from, acc, 1.0f, 1.0f, lane);
            rest += from[DB * 1024 + lane];
        }
    }
    if (BIAS) rest += attn_other_half(rest);
    if (!there) return;
    const float log_z = BIAS ? *(const volatile float*)(stat + 3 * a.stat_size) + attn_p_up<E>() : 0.0f, inv = BIAS ? attn_exp2(-log_z) : 1.0f;
    if (half == 0) { stat[0] = __builtin_fmaf(lse, ATTN_LOG2E, log_z) - attn_p_up<E>(); stat[a.stat_size] = BIAS ? __builtin_fmaf(rest, -inv, -delta) : -delta; }
    if (a.gq) attn_write_row<E, DP>(a.gq + ((int64_t)row * a.heads + head) * a.dim, acc, a.scale * inv, a.dim, half, attn_whole(a.gq, a.dim));
}

// ---- backward: gradients of the keys, the values and the bias table ----------------------------------------------------------
// A block owns 128 keys of one key head and walks the queries of the heads of its group from there on: the sums over
// shared heads are made in registers, in a fixed order.  Where that makes too few blocks for the chip, the heads and then
// the queries are shared out among several blocks, whose sums a second kernel adds up, in a fixed order too.
//
// Both sums, the keys and the values of 32 rows of 128 elements take 192 registers of a wave and leave no room for a second wave on
// its SIMD above 64 elements a head (16 bits): one wave there is limited by what it can issue (8192 tokens, 16 heads of 128:
// 416 us = 531 TFLOP/s; of 64, with two waves, 223 us = 495).  Two waves that share the work, one for each sum and both making P, take
// 406, and more for the bias; the values in LDS, 475.
__host__ __device__ inline int attn_corner(int max_distance) { return 16 * 33 + max_distance + 63; }      // floats of a wave
// Statistics of the 32 rows of a tile, two or (with a bias) four of each.  A wave brings one of them, 4 bytes a lane, twice over; where there
// are two, two waves bring the same: all count the same loads.
template <bool BIAS> constexpr int attn_stats() { return BIAS ? 4 : 2; }
constexpr int ATTN_STAT_BYTES = 256;
template <class E, int DP, bool BIAS>
__global__ __launch_bounds__(ATTN_THREADS, sizeof(E) == 2 && DP <= 64 ? 2 : 1) void attn_grad_key_kernel(const AttnArgs<E> a, int tiles, int stages) {
    using T = AttnType<E>;
    using L = AttnTile<E, DP>;
    constexpr int BM = 32, DB = DP / 32, KS = DP / 16, BYTES = BM * L::PITCH, PER = 2 * AttnStage<E, DP, BM, ATTN_WAVES>::N + 1;
    constexpr int PLACE = 2 * BYTES + attn_stats<BIAS>() * ATTN_STAT_BYTES;      // queries, gradients of the output, and their statistics
    extern __shared__ __attribute__((aligned(512))) char lds[];
    __shared__ int span[16];
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const typename L::Lane at(lane);
    float* const by_distance = (float*)(lds + stages * PLACE);   // (BIAS)
    // (its gradient) half a tile of dS of this wave, and its sums of dS for every distance
    float* const corner = by_distance + a.max_distance + 1 + wave * attn_corner(a.max_distance), *const on_distance = corner + 16 * 33;
    const int kv_heads = a.heads / a.group, parts = a.head_parts * a.query_parts;
    int tile, kv;
    attn_place(blockIdx.x, tiles, kv_heads * parts, false, tile, kv);
    const int part = kv % parts, query_part = part % a.query_parts;
    kv /= parts;
    const int key0 = tile * ATTN_ROWS + wave * 32, key = key0 + (lane & 31);
    int first, last;
    const bool there = attn_sequence<false>(a, key, lane, first, last);
    const AttnSpan own = attn_span(there, key, last), all = attn_span_of_block<ATTN_WAVES>(own, span, wave, lane);      // queries
    const int head0 = kv * a.group + part / a.query_parts * a.group / a.head_parts, heads = a.group / a.head_parts;
    float* const sums = BIAS && a.partial ? a.partial + ((int64_t)head0 * a.partial_tiles + (query_part * tiles + tile) * ATTN_WAVES + wave) * a.buckets : nullptr;
    const AttnWalk<BM> walk(all.lo, all.hi > all.lo ? all.hi : all.lo, all.inner, all.top);
    const int from = (int)((int64_t)walk.total * query_part / a.query_parts), upto = (int)((int64_t)walk.total * (query_part + 1) / a.query_parts);
    if (from == upto) {                            // no key of the block is in a sequence, or there are more parts than tiles
        if (BIAS && sums)
            for (int g = 0; g < heads; ++g)
                for (int b = lane; b < a.buckets; b += WAVE) sums[(int64_t)g * a.partial_tiles * a.buckets + b] = 0.0f;
        if (parts == 1) return;
    }
    const AttnStage<E, DP, BM, ATTN_WAVES> qs(a.q, wave, lane), os(a.go, wave, lane);
    if (a.dim * (int)sizeof(E) < L::PITCH) {
        for (int p = 0; p < stages; ++p) attn_clear(lds + p * PLACE, 2 * BYTES, tid, ATTN_THREADS);
        __syncthreads();
    }
    AttnRing ring(stages);
    const int plain = qs.plainly(a.q, a.dim) && os.plainly(a.go, a.dim) ? walk.nclean : 0;
    const int64_t to_next_q = (int64_t)BM * a.q.token, to_next_o = (int64_t)BM * a.go.token;
    const E *next_q, *next_o;
    const int which = wave % attn_stats<BIAS>();
    const float *const stats = a.stats + which * a.stat_size, *next_s;
    int next_head = head0, next = from;
    auto at_next = [&]() __attribute__((always_inline)) {
        const int64_t i0 = walk.at(next);
        next_q = a.q.p + (int64_t)next_head * a.q.head + i0 * a.q.token;
        next_o = a.go.p + (int64_t)next_head * a.go.head + i0 * a.go.token;
        next_s = stats + (int64_t)next_head * a.tokens + i0;
    };
    at_next();
    auto fetch = [&](int place) __attribute__((always_inline)) {
        char* const to = lds + place * PLACE;
        const uint32_t stat = attn_in_lds(to) + 2 * BYTES + which * ATTN_STAT_BYTES;
        if (next < plain) {
            qs.plain(a.q, next_q, attn_in_lds(to), wave);
            os.plain(a.go, next_o, attn_in_lds(to) + BYTES, wave);
            attn_load_lds<4>(next_s, (attn_lane() & 31) * 4, stat);
            next_q += to_next_q;
            next_o += to_next_o;
            next_s += BM;
        } else {
            const int i0 = walk.at(next);
            qs.load(a.q, next_head, i0, all.hi, a.dim, to, wave, lane);
            os.load(a.go, next_head, i0, all.hi, a.dim, to + BYTES, wave, lane);
            const int i = i0 + (lane & 31), in = i < all.hi ? i : all.hi - 1;
            attn_load_lds<4>(stats + (int64_t)next_head * a.tokens + i0, (uint32_t)(in - i0) * 4, stat);
        }
        if (++next == upto) {
            next = from;
            ++next_head;
            at_next();
        }
    };
    ring.begin((upto - from) * heads, fetch);
    const uint32_t reach = there ? (uint32_t)(last - key) : 0;       // query i sees the key if (unsigned)(i - key) < reach
    const float c = a.scale_log2;

    typename T::Frag k[KS], v[KS];
    attn_own_rows<E, DP>(a.k, kv, there ? key : 0, there, a.dim, lane, attn_sign(a.scale), k);
    attn_own_rows<E, DP>(a.v, kv, there ? key : 0, there, a.dim, lane, 1.0f, v);
    f32x16_t gk[DB], gv[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) {
        gk[d] = f32x16_t{};
        gv[d] = f32x16_t{};
    }
    const int e = attn_lifted<E>() ? attn_lift_of_rows(a, head0, heads, all, span, tid, lane, wave) : 0;
    const float by_ds = AttnLift::power(-attn_p_up<E>() - e), back = AttnLift::power(e);
    float far_sum = 0.0f;                      // of the head at hand, from max_distance on
    AttnFar far(0.0f, 1.0f);
    auto step = [&](auto kind_, int n, int place) __attribute__((always_inline)) {
        constexpr bool MASKED = decltype(kind_)::value == ATTN_MASKED, NEAR = BIAS && decltype(kind_)::value != ATTN_FAR;
        char* const here = lds + place * PLACE;
        const uint32_t qt = attn_in_lds(here), ot = qt + BYTES;
        const float* const st = (const float*)(here + 2 * BYTES) + 4 * half;       // the lane's rows: eight further on from four to four
        constexpr int NEXT = ATTN_STAT_BYTES / 4;
        const int i0 = walk.at(n), i = i0 + 4 * half;
        bool terms = false;
        if constexpr (MASKED) {
            terms = attn_look_over<E, ATTN_WAVES>(here, 2 * BYTES, span, tid, lane);
            if (i0 >= own.hi || i0 + BM <= own.lo) return;
        }
        const bool near = NEAR && (far.apart || i0 - (key0 + 31) < a.max_distance);
        f32x16_t s = attn_start(BIAS && !near ? far.start : 0.0f), dp;      // (dP - D: the product starts at -D)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4_t d = *(const f32x4_t*)(st + NEXT + 8 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) dp[4 * g + e] = d[e];
        }
#pragma unroll
        for (int x = 0; x < KS; ++x) s = T::mma(L::rows(qt, at, 0, x), k[x], s);
#pragma unroll
        for (int x = 0; x < KS; ++x) dp = T::mma(L::rows(ot, at, 0, x), v[x], dp);
        if (NEAR && near) {                    // (a row's exponents as they are to be: nothing is taken from them below)
            attn_add_bias<-1>(s, a.scale_abs, by_distance, i - key, a.max_distance);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4_t lse = *(const f32x4_t*)(st + 2 * NEXT + 8 * g), log_z = *(const f32x4_t*)(st + 3 * NEXT + 8 * g);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[4 * g + e] = __builtin_fmaf(s[4 * g + e] - lse[e], ATTN_LOG2E, -log_z[e]);
            }
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4_t lse2 = *(const f32x4_t*)(st + 8 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = 4 * g + e;
                const bool hidden = MASKED && (uint32_t)(i + e + 8 * g - key) >= reach;
                const float p = attn_exp2(NEAR && near ? s[r] : __builtin_fmaf(s[r], c, -lse2[e]));
                s[r] = hidden ? 0.0f : p;
                dp[r] = hidden ? 0.0f : attn_lifted<E>() ? p * (dp[r] * by_ds) : p * dp[r];
            }
        }
        if (MASKED && terms) {
            const auto sees = [&](int r) __attribute__((always_inline)) { return (uint32_t)(i0 + r - key) < reach; };
            const f32x16_t pw[1] = {s}, xw[1] = {dp};
            attn_add_terms<E, DP, 1>(here + BYTES, pw, gv, lane, sees);
            attn_add_terms<E, DP, 1>(here, xw, gk, lane, sees);
        } else {
            attn_add_product<E, DP>(ot, at, 0, s, gv);
            attn_add_product<E, DP>(qt, at, 0, dp, gk);
        }
        if (BIAS && sums) {
            if (!NEAR || i0 - (key0 + 31) >= a.max_distance) {
#pragma unroll
                for (int r = 0; r < 16; ++r) far_sum += dp[r];
            } else {
                // The tile of dS by diagonals - a distance has one value on each - 16 rows at a time: lane t adds up the
                // diagonal of distance i0 - key0 - 31 + t, and adds it to that distance's sum.  Fixed order throughout.
                float on = 0.0f;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int r = 0; r < 8; ++r) corner[(4 * half + (r & 3) + 8 * (r >> 2)) * 33 + (lane & 31)] = there ? dp[8 * h + r] : 0.0f;
                    __builtin_amdgcn_wave_barrier();
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int col = 16 * h + r + 31 - lane;
                        const float x = corner[r * 33 + (col & 31)];
                        on += col >= 0 && col < 32 ? x : 0.0f;
                    }
                    __builtin_amdgcn_wave_barrier();
                }
                const int d = i0 - key0 - 31 + lane;
                if (d >= 0 && lane < 63) on_distance[d] += on;
            }
        }
    };
    for (int g = 0; g < heads; ++g) {
        if (BIAS) {
            __syncthreads();                    // the table of the head before is not read any more
            attn_bias_by_distance(a, head0 + g, by_distance, tid, ATTN_THREADS);
            far = AttnFar(attn_bias(a, head0 + g, a.buckets - 1), a.scale_abs);
            if (sums)
                for (int n = lane; n < a.max_distance + 63; n += WAVE) on_distance[n] = 0.0f;
        }
        auto turn = [&](auto kind, int n) __attribute__((always_inline)) {
            attn_arrived<PER>(ring);
            ring.refill(fetch);
            step(kind, n, ring.at);
            ring.done();
        };
        const int clean = upto < walk.nclean ? upto : walk.nclean;
        int n = from;
        if constexpr (BIAS && DP <= 64) {           // (queries walk away from the keys: near tiles come first)
            const int beyond = far.apart ? clean : walk.nclean - attn_tiles_beyond(walk.dirty - BM - (tile * ATTN_ROWS + ATTN_ROWS - 1 + a.max_distance), BM, walk.nclean);
            for (; n < clean && n < beyond; ++n) turn(AttnKind<ATTN_CLEAN>{}, n);
            for (; n < clean; ++n) turn(AttnKind<ATTN_FAR>{}, n);
        } else {
            for (; n < clean; ++n) turn(AttnKind<ATTN_CLEAN>{}, n);
        }
        for (; n < upto; ++n) turn(AttnKind<ATTN_MASKED>{}, n);
        if (BIAS && sums && from < upto) {
            far_sum = there ? far_sum : 0.0f;   // (a column without a key is masked in the tiles of the second loop only)
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) far_sum += __shfl_xor(far_sum, d, WAVE);
            for (int b = lane; b < a.buckets; b += WAVE) {       // a bucket's distances, in order
                const int begins = b <= a.exact_to ? b : (int)a.borders[b - a.exact_to - 1];
                const int ends = b + 1 == a.buckets ? a.max_distance + 63 : b + 1 <= a.exact_to ? b + 1 : (int)a.borders[b - a.exact_to];
                float x = b + 1 == a.buckets ? far_sum : 0.0f;
                for (int n = begins; n < ends; ++n) x += on_distance[n];
                sums[(int64_t)g * a.partial_tiles * a.buckets + b] = attn_lifted<E>() ? x * back : x;
            }
            far_sum = 0.0f;
        }
    }
    if (!there) return;
    const float by_k = attn_lifted<E>() ? a.scale * back : a.scale, by_v = attn_lifted<E>() ? AttnLift::power(-14) : 1.0f;
    const int64_t out = ((int64_t)key * kv_heads + kv) * a.dim, size = (int64_t)a.tokens * kv_heads * a.dim;
    if (parts > 1) attn_write_row<float, DP>(a.part_k + part * size + out, gk, by_k, a.dim, half, a.dim % 4 == 0);
    else if (a.gk) attn_write_row<E, DP>(a.gk + out, gk, by_k, a.dim, half, attn_whole(a.gk, a.dim));
    if (parts > 1) attn_write_row<float, DP>(a.part_v + part * size + out, gv, by_v, a.dim, half, a.dim % 4 == 0);
    else if (a.gv) attn_write_row<E, DP>(a.gv + out, gv, by_v, a.dim, half, attn_whole(a.gv, a.dim));
}

// dk and dv from their parts, in order; rows that no sequence holds are left as they are
template <class E, int N>
__global__ __launch_bounds__(ATTN_THREADS) void attn_join_parts_kernel(const AttnArgs<E> a, int parts, int64_t units, int row) {
    const int64_t u = (int64_t)blockIdx.x * ATTN_THREADS + threadIdx.x;
    if (u >= units) return;
    const int token = (int)(u / (row / N));
    if (token < a.offsets[0] || token >= a.offsets[a.sequences]) return;
    const float* const from = blockIdx.y ? a.part_v : a.part_k;
    E* const to = blockIdx.y ? a.gv : a.gk;
    if (!to) return;
    float x[N] = {};
    for (int p = 0; p < parts; ++p) {
        float y[N];
        __builtin_memcpy(y, __builtin_assume_aligned(from + ((int64_t)p * units + u) * N, N * 4), sizeof(y));
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] += y[e];
    }
    E z[N];
#pragma unroll
    for (int e = 0; e < N; ++e) z[e] = AttnType<E>::put(x[e]);
    __builtin_memcpy(__builtin_assume_aligned(to + u * N, N * sizeof(E)), z, sizeof(z));
}

// dtable[b][h]: the partial sums of the key tiles, in their order
template <class E>
__global__ __launch_bounds__(ATTN_THREADS) void attn_grad_table_kernel(const float* partial, int tiles, int buckets, int heads, E* table) {
    const int b = blockIdx.x, h = blockIdx.y;
    __shared__ float sum[ATTN_THREADS / WAVE];
    float x = 0.0f;
    for (int t = threadIdx.x; t < tiles; t += ATTN_THREADS) x += partial[((int64_t)h * tiles + t) * buckets + b];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d, WAVE);
    if (threadIdx.x % WAVE == 0) sum[threadIdx.x / WAVE] = x;
    __syncthreads();
    if (threadIdx.x == 0) table[(int64_t)b * heads + h] = AttnType<E>::put((sum[0] + sum[1]) + (sum[2] + sum[3]));
}

// ---- host ----------------------------------------------------------------------------------------------------------------
// attention.hip: least whole distance n with (n / E)^M >= (X / E)^m for m = 1 .. M - 1, exactly
bool attn_borders(int buckets, int max_distance, uint16_t* borders);

template <class E>
inline bool attn_view(AttnView<E>& v, const void* base, const size_t* strides, size_t offset, int dim) {
    v.p = (const E*)base + offset;
    v.token = (int64_t)strides[0];
    v.head = (int64_t)strides[1];
    v.elem = (int64_t)strides[2];
    constexpr size_t N = AttnType<E>::CHUNK;
    // a tile of 64 rows is addressed with 32-bit offsets
    v.vec = (strides[2] == 1 || dim == 1) && dim % N == 0 && strides[0] % N == 0 && strides[1] % N == 0 && (uintptr_t)v.p % 16 == 0 && strides[0] < (1u << 23);
    return true;
}

// metadata: tokens, heads, kv_heads, dim, sequences, buckets, max_distance | q, k, v strides | q, k, v offsets
template <class E>
inline bool attn_arguments(AttnArgs<E>& a, const size_t* md, const int32_t* offsets, const E* q, const E* k, const E* v, const E* table, float scale) {
    const bool some = !md || md[0] != 0;        // (tensors of no tokens have no address)
    if (!md || !offsets || (some && (!q || !k || !v))) { set_status(ERR_INVALID, "attention: null argument"); return false; }
    const size_t tokens = md[0], heads = md[1], kv = md[2], dim = md[3], sequences = md[4];
    if (heads == 0 || kv == 0 || dim == 0 || heads % kv != 0) { set_status(ERR_INVALID, "attention: heads must be a multiple of kv_heads, and dim positive"); return false; }
    if (dim > (size_t)ATTN_MAX_DIM) { set_status(ERR_UNSUPPORTED, "attention: head dimension above 128"); return false; }
    if (tokens >= (1ull << 31) - 1024 || sequences >= (1ull << 31) - 1024 || heads > 65535) { set_status(ERR_TOO_LARGE, "attention: too many tokens, sequences or heads"); return false; }
    if (((tokens + ATTN_ROWS - 1) / ATTN_ROWS) * heads * ATTN_THREADS >= (1ull << 32)) { set_status(ERR_TOO_LARGE, "attention: too many tiles"); return false; }
    std::memset((void*)&a, 0, sizeof(a));
    attn_view(a.q, q, md + 7, md[16], (int)dim);
    attn_view(a.k, k, md + 10, md[17], (int)dim);
    attn_view(a.v, v, md + 13, md[18], (int)dim);
    a.offsets = offsets;
    a.table = table;
    a.tokens = (int32_t)tokens;
    a.heads = (int32_t)heads;
    a.group = (int32_t)(heads / kv);
    a.dim = (int32_t)dim;
    a.sequences = (int32_t)sequences;
    a.scale = scale;
    a.scale_abs = scale == 0.0f ? 1.0f : std::fabs(scale);
    a.scale_log2 = a.scale_abs * ATTN_LOG2E;
    if (table) {
        const size_t buckets = md[5], distance = md[6];
        if (buckets < 2 || buckets > (size_t)ATTN_MAX_BUCKETS) { set_status(ERR_UNSUPPORTED, "attention: a bias takes 2 to 256 buckets"); return false; }
        if (distance <= buckets / 2 || distance > (size_t)ATTN_MAX_DISTANCE) { set_status(ERR_UNSUPPORTED, "attention: max_distance lies above buckets / 2 and up to 4096"); return false; }
        a.buckets = (int32_t)buckets;
        a.exact_to = (int32_t)(buckets / 2);
        a.max_distance = (int32_t)distance;
        if (!attn_borders((int)buckets, (int)distance, a.borders)) return false;
    }
    if (tokens == 0 || sequences == 0) return true;
    a.flag = index_flag();
    return a.flag != nullptr;
}

// more than 64 KB of LDS has to be asked for, once for each kernel and device
inline bool attn_lds(const void* kernel, size_t bytes, uint64_t& asked) {
    if (bytes <= 60 * 1024) return true;
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) { set_status(ERR_INVALID, "attention: bad device"); return false; }
    if (asked >> dev & 1) return true;
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024 - 1024);
    if (e != hipSuccess) { set_status(ERR_LAUNCH, "attention: LDS size", (int)e); return false; }
    asked |= 1ull << dev;
    return true;
}

// Places of a ring: as many as help (four) and fit beside `rest`, `blocks` sharing a CU's LDS, `rings` a block's.
inline int attn_stages(size_t place, size_t rest, int rings, int blocks) {
    const int64_t room = 160 * 1024 / blocks - 512 - (int64_t)rest, n = room / (int64_t)(place * rings);
    return n >= 4 ? 4 : n >= 3 ? 3 : n >= 2 || blocks == 1 ? 2 : attn_stages(place, rest, rings, 1);
}
template <int KG, class Kernel, class E>
inline void attn_row_launch(Kernel* kernel, const AttnArgs<E>& a, size_t place, uint64_t& asked, const char* what) {
    const int rows = 32 * attn_row_waves<KG>(), tiles = (a.tokens + rows - 1) / rows;
    const unsigned blocks = (unsigned)(tiles * a.heads);
    const size_t rest = a.table ? ((size_t)a.max_distance + 1) * 4 : 0;
    const int stages = attn_stages(place, rest, KG, KG > 1 || blocks <= 256 ? 1 : 2);
    const size_t lds = KG * stages * place + rest;
    if (!attn_lds((const void*)kernel, lds, asked)) return;
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(64 * attn_row_waves<KG>() * KG), lds, stream(), a, tiles, stages);
    MXH_LAUNCH_CHECK(what);
}
// Up to two blocks for every CU, the time is that of the longest walks: two groups of waves share each (one block of 512
// threads to a CU).  Beyond, they are ahead no more: 4096 tokens in one sequence, 16 heads of 128 (512 blocks): 93 against 110 us
// forward, 32 heads: 185 against 161 us.  With less than three blocks for four CUs, four groups share the walks of half as many
// rows: f32, 1024 tokens, 8 heads of 64 with a bias (64 blocks) 47 -> 31 us forward, 65 -> 41 us dq, f16, 1802 tokens, 12 heads of 80 (180
// blocks) 34 -> 29 and 40 -> 33 us; with 256 blocks they lose: bf16, 2000 tokens, 16 heads of 64: 32 -> 40 us.
// f32 heads above 64 take too many registers for either.  At 128 elements (16 bits) four groups read up to 29 registers back from memory and
// are ahead all the same: 1024 tokens, 16 heads (128 blocks): 25 -> 24 us forward, 34 -> 28 dq; 2048 tokens, 8 heads: 40 -> 36, 54 -> 41.
// At 192 blocks, where twice as many of half the rows are one and a half for a CU, it goes by the walks: 2048 tokens, 12 heads of 96:
// 40 -> 37, 48 -> 43; 1024 tokens, 24 heads: 25 -> 28, 31 -> 34 (of 128: 41 -> 43, 55 -> 50 and 26 -> 33, 36 -> 41).
template <class E, int DP>
inline int attn_groups(const AttnArgs<E>& a) {
    const int64_t blocks = (int64_t)((a.tokens + ATTN_ROWS - 1) / ATTN_ROWS) * a.heads;
    return (sizeof(E) == 4 && DP > 64) || blocks > 512 ? 1 : blocks > 192 ? 2 : 4;
}

template <class E, int DP, bool BIAS, int KG>
inline void attn_forward_groups(const AttnArgs<E>& a) {
    static uint64_t asked = 0;
    attn_row_launch<KG>(attn_forward_kernel<E, DP, BIAS, KG>, a, 2 * attn_tile_bytes<E, DP>(attn_keys<E, DP, KG>()), asked, "attention");
}
template <class E, int DP, bool BIAS, int KG>
inline void attn_query_groups(const AttnArgs<E>& a) {
    static uint64_t asked = 0;
    attn_row_launch<KG>(attn_grad_query_kernel<E, DP, BIAS, KG>, a, 2 * attn_tile_bytes<E, DP>(attn_grad_keys<E, DP, KG>()), asked, "attention_backward (queries)");
}
template <class E, int DP, bool BIAS>
inline void attn_forward_launch(const AttnArgs<E>& a) {
    if constexpr (!(sizeof(E) == 4 && DP > 64)) {
        if (attn_groups<E, DP>(a) == 4) return attn_forward_groups<E, DP, BIAS, 4>(a);
        if (attn_groups<E, DP>(a) == 2) return attn_forward_groups<E, DP, BIAS, 2>(a);
    }
    attn_forward_groups<E, DP, BIAS, 1>(a);
}
template <class E, int DP, bool BIAS>
inline void attn_query_launch(const AttnArgs<E>& a) {
    if constexpr (!(sizeof(E) == 4 && DP > 64)) {
        if (attn_groups<E, DP>(a) == 4) return attn_query_groups<E, DP, BIAS, 4>(a);
        if (attn_groups<E, DP>(a) == 2) return attn_query_groups<E, DP, BIAS, 2>(a);
    }
    attn_query_groups<E, DP, BIAS, 1>(a);
}
template <class E, int DP, bool BIAS>
inline void attn_backward_launch(const AttnArgs<E>& a, E* grad_table) {
    static uint64_t asked_k = 0;
    const int tiles = (a.tokens + ATTN_ROWS - 1) / ATTN_ROWS, kv = a.heads / a.group;
    const size_t bias = BIAS ? ((size_t)a.max_distance + 1) * 4 : 0;
    attn_query_launch<E, DP, BIAS>(a);
    if (a.gk || a.gv || grad_table) {
        const size_t place = 2 * attn_tile_bytes<E, DP>(32) + attn_stats<BIAS>() * ATTN_STAT_BYTES, rest = bias + (BIAS && grad_table ? (size_t)ATTN_WAVES * attn_corner(a.max_distance) * 4 : 0);
        const int parts = a.head_parts * a.query_parts;
        const unsigned blocks = (unsigned)(tiles * kv * parts);
        const int stages = attn_stages(place, rest, 1, sizeof(E) == 2 && DP <= 64 && blocks > 256 ? 2 : 1);
        auto* kernel = attn_grad_key_kernel<E, DP, BIAS>;
        if (!attn_lds((const void*)kernel, stages * place + rest, asked_k)) return;
        hipLaunchKernelGGL(kernel, dim3(blocks), dim3(ATTN_THREADS), stages * place + rest, stream(), a, tiles, stages);
        MXH_LAUNCH_CHECK("attention_backward (keys)");
        if (parts > 1 && (a.gk || a.gv)) {
            const int row = kv * a.dim;
            const bool whole = row % 4 == 0 && (uintptr_t)a.gk % (4 * sizeof(E)) == 0 && (uintptr_t)a.gv % (4 * sizeof(E)) == 0;
            const int64_t units = (int64_t)a.tokens * row / (whole ? 4 : 1);
            const dim3 grid(cdiv((size_t)units, (size_t)ATTN_THREADS), 2);
            if (whole) hipLaunchKernelGGL((attn_join_parts_kernel<E, 4>), grid, dim3(ATTN_THREADS), 0, stream(), a, parts, units, row);
            else hipLaunchKernelGGL((attn_join_parts_kernel<E, 1>), grid, dim3(ATTN_THREADS), 0, stream(), a, parts, units, row);
            MXH_LAUNCH_CHECK("attention_backward (parts)");
        }
    }
    if (grad_table) {
        hipLaunchKernelGGL(attn_grad_table_kernel<E>, dim3((unsigned)a.buckets, (unsigned)a.heads), dim3(ATTN_THREADS), 0, stream(), a.partial, a.partial_tiles, a.buckets, a.heads, grad_table);
        MXH_LAUNCH_CHECK("attention_backward (bias)");
    }
}
// the head dimension is padded with zeros to 32, 64, 96 or 128
template <class E, class F>
inline void attn_by_dim(const AttnArgs<E>& a, F&& f) {
    if (a.dim <= 32) f(std::integral_constant<int, 32>{});
    else if (a.dim <= 64) f(std::integral_constant<int, 64>{});
    else if (a.dim <= 96) f(std::integral_constant<int, 96>{});
    else f(std::integral_constant<int, 128>{});
}

template <class E>
inline void attention_entry(const size_t* md, const int32_t* offsets, const E* q, const E* k, const E* v, const E* table, float scale, E* out, float* lse) {
    AttnArgs<E> a;
    if ((!out || !lse) && !(md && md[0] == 0)) { set_status(ERR_INVALID, "attention: null output"); return; }
    if (!attn_arguments(a, md, offsets, q, k, v, table, scale)) return;
    if (a.tokens == 0 || a.sequences == 0) return;
    a.out = out;
    a.lse = lse;
    attn_by_dim(a, [&](auto dp) {
        if (table) attn_forward_launch<E, decltype(dp)::value, true>(a);
        else attn_forward_launch<E, decltype(dp)::value, false>(a);
    });
}

template <class E>
inline void attention_backward_entry(const size_t* md, const int32_t* offsets, const E* q, const E* k, const E* v, const E* table, float scale, const E* out,
                                     const float* lse, const E* grad_out, E* gq, E* gk, E* gv, E* grad_table) {
    AttnArgs<E> a;
    if ((!out || !lse || !grad_out) && !(md && md[0] == 0)) { set_status(ERR_INVALID, "attention_backward: null argument"); return; }
    if (grad_table && !table) { set_status(ERR_INVALID, "attention_backward: the gradient of a bias that was not given"); return; }
    if (!attn_arguments(a, md, offsets, q, k, v, table, scale)) return;
    if (!gq && !gk && !gv && !grad_table) return;
    const size_t rows[3] = {(size_t)a.heads * a.dim, (size_t)a.dim, 1};
    attn_view(a.o, out, rows, 0, a.dim);
    attn_view(a.go, grad_out, rows, 0, a.dim);
    a.lse = (float*)lse;
    a.gq = gq;
    a.gk = gk;
    a.gv = gv;
    if (a.tokens == 0 || a.sequences == 0) {        // no pair: the table's gradient is zero
        if (!grad_table) return;
        hipLaunchKernelGGL(attn_grad_table_kernel<E>, dim3((unsigned)a.buckets, (unsigned)a.heads), dim3(ATTN_THREADS), 0, stream(), (const float*)nullptr, 0, a.buckets, a.heads, grad_table);
        MXH_LAUNCH_CHECK("attention_backward (bias)");
        return;
    }
    // parts of the kernel of the keys: until there are two blocks for every CU, first the heads of a group, then the queries
    // (eight tiles of them at least)
    const size_t tiles = cdiv((size_t)a.tokens, (size_t)ATTN_ROWS), kv = (size_t)(a.heads / a.group);
    a.head_parts = a.query_parts = 1;
    while (a.head_parts < a.group && (tiles * kv * a.head_parts < 512 || a.group % a.head_parts != 0)) ++a.head_parts;
    while (tiles * kv * a.head_parts * a.query_parts < 512 && (size_t)a.tokens / 32 / a.query_parts >= 16) a.query_parts *= 2;
    const int parts = a.head_parts * a.query_parts;
    const size_t stats = ((size_t)a.heads * a.tokens + 63) / 64 * 64, sums = parts > 1 ? ((size_t)a.tokens * kv * a.dim + 63) / 64 * 64 * parts : 0;
    const size_t all_stats = stats * (table ? 4 : 2), lifts = attn_lifted<E>() ? (size_t)a.heads * cdiv((size_t)a.tokens, 32) * 4 : 0;
    a.partial_tiles = (int)(ATTN_WAVES * tiles) * a.query_parts;
    const size_t partials = grad_table ? (size_t)a.heads * a.partial_tiles * a.buckets : 0;
    a.stats = (float*)scratch((all_stats + 2 * sums + partials + lifts) * sizeof(float));
    if (!a.stats) return;
    a.stat_size = (int64_t)stats;
    a.part_k = a.stats + all_stats;
    a.part_v = a.part_k + sums;
    a.partial = grad_table ? a.part_v + sums : nullptr;
    a.lifts = (int32_t*)(a.part_v + sums + partials);
    attn_by_dim(a, [&](auto dp) {
        if (table) attn_backward_launch<E, decltype(dp)::value, true>(a, grad_table);
        else attn_backward_launch<E, decltype(dp)::value, false>(a, grad_table);
    });
}

#define MXH_ATTENTION(E, S)                                                                                                                          \
    extern "C" void hip_attention_##S(const size_t* metadata, const int32_t* offsets, const E* query, const E* key, const E* value, const E* bias,   \
                                      float scale, E* output, float* lse) { MXH_API;                                                                 \
        ::mxh::attention_entry<E>(metadata, offsets, query, key, value, bias, scale, output, lse);                                                   \
    }                                                                                                                                                \
    extern "C" void hip_attention_backward_##S(const size_t* metadata, const int32_t* offsets, const E* query, const E* key, const E* value,         \
                                               const E* bias, float scale, const E* output, const float* lse, const E* grad_output, E* grad_query,   \
                                               E* grad_key, E* grad_value, E* grad_bias) { MXH_API;                                                  \
        ::mxh::attention_backward_entry<E>(metadata, offsets, query, key, value, bias, scale, output, lse, grad_output, grad_query, grad_key,        \
                                           grad_value, grad_bias);                                                                                   \
    }

}  // namespace mxh
