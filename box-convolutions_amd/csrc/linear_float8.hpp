// The pointwise product of rows in 8-bit blocks of 128 (float8_blocks.hpp): y = act(x W^T + bias + residual), both operands K-major.
// The matrix instructions multiply by the blocks' powers of two themselves: each lane gives one exponent for the 32 values that it holds
// of a row.
#pragma once

#include "float8_blocks.hpp"
#include "linear_wide.hpp"

namespace boxconv {

namespace {

// One operand: [extent] rows of `blocks` blocks of codes, and `padded` exponents each.
struct Coded {
    const uint8_t *codes, *exponents;
    int64_t extent;
    int blocks, padded;
};

// 32 codes of a row: a lane's share of 64 values of k.
struct Codes32 { Chunk lo, hi; };

// The 8-bit instructions cut every product of 8 neighbouring k down to a multiple of 2^-13 of the largest of them before they add (found
// with products of one large and one small pair: one 2^13 times smaller is kept, one 2^14 times smaller is lost, from the ninth k on nothing
// is). That is 1e-5 to 4e-5 of a sum of random signs, far below half a step of the 16-bit types. Results in float32 take the bfloat16
// instructions instead, at half the rate: codes and powers of two fit that type, and its products add up in float32.
typedef int Eight __attribute__((ext_vector_type(8)));
template <class T>
__device__ __forceinline__ Acc16 multiply_add8(const Codes32& b, int eb, const Codes32& a, int ea, Acc16 c) {
    typedef __bf16 Pair __attribute__((ext_vector_type(2)));
    typedef __bf16 Run __attribute__((ext_vector_type(8)));
    if constexpr (sizeof(T) == 2) {
        const auto join = [](const Codes32& v) { return __builtin_bit_cast(Eight, v); };
        return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(join(b), join(a), c, 0, 0, 0, eb, 0, ea);
    } else {
        const auto wide = [](const Codes32& v, int e, int i) {             // eight codes as bfloat16
            const float power = __builtin_bit_cast(float, (static_cast<unsigned>(e) & 255) << 23);
            const Chunk from = i < 2 ? v.lo : v.hi;
            Run out;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const unsigned word = from[i % 2 * 2 + j / 2];
                const Pair two = j % 2 == 0 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, power, false) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, power, true);
                out[2 * j] = two[0];
                out[2 * j + 1] = two[1];
            }
            return out;
        };
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wide(b, eb, i), wide(a, ea, i), c, 0, 0, 0);
        return c;
    }
}

// A byte as an operand's element, for the tiles and the feed of the wide kernels.
struct Code { uint8_t bits; };
template <> struct Vec<Code> { static constexpr int kLen = 16; typedef uint8_t Type __attribute__((ext_vector_type(16), aligned(1))); };

// 4 bytes per lane from `offset` bytes into a descriptor's memory to LDS at `to` + 4 * lane.
__device__ __forceinline__ void word_to_lds(Descriptor d, unsigned offset, unsigned to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(to), "v"(offset), "s"(d) : "m0");
}

// TM x TN tile by WM x WN waves, each with (TM/WM) x (TN/WN), as in product_wide_kernel: two stages of LDS, each a block of 128 codes of every
// row. A block is two steps of 64 values of k. The barrier stands between them: the second step's fragments are in registers by then, so the
// stage takes the block after next, whose loads go out one at a time between the second step's products. Exponents come four blocks at a time, a
// word of every row, into a ring of their own; a lane keeps the words of its rows and shifts them by a byte from block to block.
template <class T, int TM, int TN, int WM, int WN>
__global__ void __launch_bounds__(WM * WN * 64)
product_float8_kernel(Coded a, Coded b, Tail<T> tail, int part_blocks, unsigned tiles_m, unsigned tiles_n) {
    typedef TileShape<Code, true, TM, 8> SA;
    typedef TileShape<Code, true, TN, 8> SB;
    constexpr int THREADS = WM * WN * 64, FM = TM / WM / 32, FN = TN / WN / 32;
    constexpr int kStage = SA::kChunks + SB::kChunks;
    static_assert(THREADS >= TM + TN && TM % 64 == 0 && SA::KT == kBlock, "a thread per row of exponents, whole waves of them; a block a stage");
    extern __shared__ Chunk stages[];
    unsigned* const words = reinterpret_cast<unsigned*>(stages + kRing * kStage);          // [2][TM + TN]
    unsigned tm, tn, part;
    tile_of(tiles_m, tiles_n, tm, tn, part);
    const int64_t m0 = static_cast<int64_t>(tm) * TM, n0 = static_cast<int64_t>(tn) * TN;
    const int first = static_cast<int>(part) * part_blocks, steps = min(a.blocks - first, part_blocks);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), wm = wave / WN * (TM / WM), wn = wave % WN * (TN / WN), l = threadIdx.x % 64;
    Acc16 acc[FN][FM] = {};
    typedef Feed<Code, true, TM, THREADS, false> FeedA;
    typedef Feed<Code, true, TN, THREADS, true> FeedB;
    FeedA fa;
    FeedB fb;
    const int64_t row_bytes = static_cast<int64_t>(a.blocks) * kBlock;
    fa.start({reinterpret_cast<const Code*>(a.codes), row_bytes, a.extent, row_bytes}, m0, static_cast<int64_t>(first) * kBlock);
    fb.start({reinterpret_cast<const Code*>(b.codes), row_bytes, b.extent, row_bytes}, n0, static_cast<int64_t>(first) * kBlock);
    // the exponents of this wave's 64 rows of the tile
    const bool of_a = wave * 64 < TM;
    const int64_t row0 = of_a ? m0 + wave * 64 : n0 + wave * 64 - TM, rows = (of_a ? a.extent : b.extent) - row0;
    const uint64_t at = reinterpret_cast<uint64_t>((of_a ? a.exponents : b.exponents) + row0 * a.padded);
    const auto scalar = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    const Descriptor dw = {scalar(static_cast<int>(at)), scalar(static_cast<int>(at >> 32) & 0xffff),
                           scalar(rows <= 0 ? 0 : static_cast<int>(min<int64_t>(rows, 64)) * a.padded), 0x00020000};
    const auto load_words = [&](int group) {                   // (beyond the end: zeros, which nobody uses)
        if (wave * 64 < TM + TN)
            word_to_lds(dw, 4 * group < a.padded ? static_cast<unsigned>(l * a.padded + 4 * group) : kNowhere,
                        scalar(static_cast<int>(reinterpret_cast<uintptr_t>((LdsVoid)(words + (group & 1) * (TM + TN)))) + wave * 256));
    };
    Descriptor da, db;
    const auto load = [&](int s, int i) {
        const Chunk* tile = stages + s % kRing * kStage;
        const int k_left = (steps - s) * kBlock;
        if (i == 0) da = fa.next();
        if (i == FeedA::N) db = fb.next();
        if (i < FeedA::N) fa.fetch(da, i, tile, k_left);
        else fb.fetch(db, i - FeedA::N, tile + SA::kChunks, k_left);
    };
    // Fragments of the step at hand and of the next: of A in two sets, of B in one and a spare, which takes the next step's last fragment while
    // every other replaces its own (two sets of B as well do not fit the registers of 256 x 256 tiles).
    Codes32 xa[2][FM], xb[FN + 1];
    const auto take = [&](int s, int h, int f) {
        const Chunk* tile = stages + s % kRing * kStage;
        return f < FM ? Codes32{fragment<Code, true, TM, 8, false>(tile, wm + 32 * f, 2 * h), fragment<Code, true, TM, 8, false>(tile, wm + 32 * f, 2 * h + 1)}
                      : Codes32{fragment<Code, true, TN, 8, true>(tile + SA::kChunks, wn + 32 * (f - FM), 2 * h),
                                fragment<Code, true, TN, 8, true>(tile + SA::kChunks, wn + 32 * (f - FM), 2 * h + 1)};
    };
    const auto slot = [](int h, int j) { return j < FN - 1 ? j : FN - 1 + h; };
    unsigned ea[FM], eb[FN];
    constexpr int kLoads = FeedA::N + FeedB::N, kProducts = FM * FN;
    // step h: its products, and between them the loads of stage `to` (none: -1) and the reads of the other step, of stage `from`
    const auto step = [&](int h, int from, int to) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int p = 0; p < kProducts; ++p) {
            if (p < FM) xa[h ^ 1][p] = take(from, h ^ 1, p);
            if (p == min(1, kProducts - 1)) xb[slot(h ^ 1, FN - 1)] = take(from, h ^ 1, FM + FN - 1);
            if (p % FM == 0 && p > 0) xb[p / FM - 1] = take(from, h ^ 1, FM + p / FM - 1);
            if (to >= 0) {
#pragma unroll
                for (int i = p * kLoads / kProducts; i < (p + 1) * kLoads / kProducts; ++i) load(to, i);
            }
            acc[p / FM][p % FM] = multiply_add8<T>(xb[slot(h, p / FM)], eb[p / FM], xa[h][p % FM], ea[p % FM], acc[p / FM][p % FM]);
            asm volatile("" : "+v"(acc[p / FM][p % FM]));      // (keeps the product here: it would be moved behind all loads and reads of the stage, and spill)
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    if (steps > 0) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) load(0, i);
        load_words(first / 4);
        settle<0>();
#pragma unroll
        for (int i = 0; i < FM; ++i) xa[0][i] = take(0, 0, i);
#pragma unroll
        for (int i = 0; i < FN; ++i) xb[slot(0, i)] = take(0, 0, FM + i);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) load(1, i);
    }
    for (int s = 0; s < steps; ++s) {
        if (s % 4 == 0) {
            const int group = (first + s) / 4;
            const unsigned* from = words + (group & 1) * (TM + TN);
#pragma unroll
            for (int i = 0; i < FM; ++i) ea[i] = from[wm + 32 * i + l % 32];
#pragma unroll
            for (int i = 0; i < FN; ++i) eb[i] = from[TM + wn + 32 * i + column_of(l % 32)];
            load_words(group + 1);
        }
        step(0, s, -1);
        settle<0>();                                           // stage s + 1 has landed, and the rest of this one is in registers
        step(1, s + 1, s + 2);
#pragma unroll
        for (int i = 0; i < FM; ++i) ea[i] >>= 8;
#pragma unroll
        for (int i = 0; i < FN; ++i) eb[i] >>= 8;
    }
    settle<0>();                                               // every wave's loads have landed and its fragments are read: the LDS is free
    static_assert(WM * WN * 256 * FN <= kRing * kStage, "each wave turns its sums in a part of the stages");
    store_blocks<T, FN, FM>(tail, acc, m0 + wm, n0 + wn, part, stages + wave * 256 * FN);
}

}  // namespace

}  // namespace boxconv
