// The pointwise product of rows in 8-bit blocks of 128 (float8_blocks.hpp): y = act(x W^T + bias + residual), both operands K-major.
// The matrix instructions multiply by the blocks' powers of two themselves: each lane gives one exponent for the 32 values that it holds
// of a row.
#pragma once

#include <type_traits>

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

// The 8-bit instructions cut every product of 8 neighbouring k down, towards zero, to a multiple of 2^-13 of the largest of them before they add (found
// with products of one large and one small pair: one 2^13 times smaller is kept, one 2^14 times smaller is lost, of either sign, from the ninth k on nothing
// is). Measured against 64 bits: 1.5e-5 to 4e-5 of a sum of random signs, -3e-6 of a sum of one sign (normal values, K 64 to 4096), by a model of the cut
// -1e-5 to -1e-4 where channels differ by factors of e to e^2; at worst 7 * 2^-13 of each group's largest product. Half a step of the 16-bit types is 2^-9 to
// 2^-8 and 2^-12 to 2^-11, but of the result: where large products cancel, what is left of small ones beside them can be lost. 16-bit results take these
// instructions all the same: their operands were rounded to 2^-4. Results in float32 take the bfloat16 instructions instead, at half the rate or less: codes and
// powers of two fit that type, and its products add up in float32.
typedef int Eight __attribute__((ext_vector_type(8)));
typedef __bf16 Run __attribute__((ext_vector_type(8)));
typedef float Acc4 __attribute__((ext_vector_type(4)));

// Codes 8 i to 8 i + 7 times their block's power.
__device__ __forceinline__ Run as_bfloat16(const Codes32& v, int exponent, int i) {
    typedef __bf16 Pair __attribute__((ext_vector_type(2)));
    const float power = __builtin_bit_cast(float, (static_cast<unsigned>(exponent) & 255) << 23);
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
}

// 32 x 32 results, 64 values of k; 16 x 16, 128. The low byte of an exponent counts.
__device__ __forceinline__ Acc16 multiply_add_scaled(const Codes32& b, int eb, const Codes32& a, int ea, Acc16 c) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(__builtin_bit_cast(Eight, b), __builtin_bit_cast(Eight, a), c, 0, 0, 0, eb, 0, ea);
}
__device__ __forceinline__ Acc4 multiply_add_scaled(const Codes32& b, int eb, const Codes32& a, int ea, Acc4 c) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(__builtin_bit_cast(Eight, b), __builtin_bit_cast(Eight, a), c, 0, 0, 0, eb, 0, ea);
}
__device__ __forceinline__ Acc16 multiply_add_decoded(const Codes32& b, int eb, const Codes32& a, int ea, Acc16 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bfloat16(b, eb, i), as_bfloat16(a, ea, i), c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ Acc4 multiply_add_decoded(const Codes32& b, int eb, const Codes32& a, int ea, Acc4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bfloat16(b, eb, i), as_bfloat16(a, ea, i), c, 0, 0, 0);
    return c;
}
// The row of the first operand that result i of a lane belongs to (its row of the second is the lane's own).
__device__ __forceinline__ int first_row(const Acc16&, int i) { return 8 * (i / 4) + threadIdx.x % 64 / 32 * 4 + i % 4; }
__device__ __forceinline__ int first_row(const Acc4&, int i) { return threadIdx.x % 64 / 16 * 4 + i; }

// bfloat16 holds every code as a normal number under the exponents 10 to 246 (2^-9 * 2^-117 to 448 * 2^119). Under others (a block with a value next to
// the type's largest has 247; 0 is no block's but that of rows beyond the operand, which are zeros) a sum is formed with the nearest of these, and multiplied
// by what is left over, a power of two. Asked once a block, and not in front of every product: 8192 x 4096 -> 2048 float32 167 to 172 us without, 172 to 176
// this way, 191 to 196 that way. (Few rows ask that way: 32 rows of 2048 -> 4096 8.3 us without, 9.2 so.)
__device__ __forceinline__ int held_exponent(int e) { return min(max(e & 255, 10), 246); }
__device__ __forceinline__ bool beyond_bfloat16(int e) { return (e & 255) != 0 && held_exponent(e) != (e & 255); }

// BEYOND (results in float32): exponents beyond those of bfloat16 too.
template <class T, bool BEYOND, class Acc>
__device__ __forceinline__ Acc multiply_add8(const Codes32& b, int eb, const Codes32& a, int ea, Acc c) {
    if constexpr (sizeof(T) == 2) return multiply_add_scaled(b, eb, a, ea, c);
    else if constexpr (!BEYOND) return multiply_add_decoded(b, eb, a, ea, c);
    else {
        int xa = held_exponent(ea), xb = held_exponent(eb);
        const int of_a = (ea & 255) - xa, of_b = (eb & 255) - xb;
        asm volatile("" : "+v"(xa), "+v"(xb));                 // (or operands would be decoded ahead of the branch that leads here)
        const Acc sum = multiply_add_decoded(b, xb, a, xa, Acc{});
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(Acc) / sizeof(float)); ++i) c[i] += ldexpf(sum[i], of_a + __shfl(of_b, first_row(c, i)));
        return c;
    }
}
// f(std::true_type()) where the wave has an exponent beyond those of bfloat16 and that matters, else f(std::false_type()).
template <class T, class F>
__device__ __forceinline__ void with_exponents(bool beyond, F f) {
    if constexpr (sizeof(T) == 4) {
        if (__builtin_expect(__any(beyond), 0)) return f(std::true_type());
    }
    f(std::false_type());
}

// A byte as an operand's element, for the tiles and the feed of the wide kernels.
struct Code { uint8_t bits; };
template <> struct Vec<Code> { static constexpr int kLen = 16; typedef uint8_t Type __attribute__((ext_vector_type(16), aligned(1))); };

// 4 bytes per lane from `offset` bytes into a descriptor's memory to LDS at `to` + 4 * lane.
__device__ __forceinline__ void word_to_lds(Descriptor d, unsigned offset, unsigned to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(to), "v"(offset), "s"(d) : "m0");
}

// TM x TN tile by WM x WN waves, each with (TM/WM) x (TN/WN), as in product_wide_kernel: RING stages of LDS (a power of two), each a block of 128
// codes of every row. A block is two steps of 64 values of k. The barrier stands between them: the second step's fragments are in registers by then, so the
// stage takes a block RING further on, whose loads go out one at a time between the second step's products. Exponents come four blocks at a time, a
// word of every row, into a ring of their own; a lane keeps the words of its rows and shifts them by a byte from block to block.
// Bound by the matrix instructions while tiles go round: 8192 x 8192 -> 8192 bfloat16 486 us (2.3 PFLOP/s; 452 at best), where a library's product with one scale
// a tensor reaches 2.6. With one tile a compute unit its first loads and its epilogue are not hidden: 8192 x 4096 -> 2048 repeated alone 61 us (2.3 PFLOP/s), with
// silu, bias and a residual 66, right behind the launch that quantizes its rows 80 to 85, a library's without them 50; 8192 x 2048 -> 4096 69, with gelu 87, behind
// the norm that writes its rows 102 to 105, a library's 65. Float32 results: 8192 x 8192 -> 8192 1.30 ms (0.85 PFLOP/s), 8192 x 4096 -> 2048 174 to 210 us. (Medians.)
// No better: parts of k that start at another block in every tile, four waves for a tile of 256 x 256.
template <class T, int TM, int TN, int WM, int WN, int RING>
__global__ void __launch_bounds__(WM * WN * 64)
product_float8_kernel(Coded a, Coded b, Tail<T> tail, int part_blocks, unsigned tiles_m, unsigned tiles_n) {
    typedef TileShape<Code, true, TM, 8> SA;
    typedef TileShape<Code, true, TN, 8> SB;
    constexpr int THREADS = WM * WN * 64, FM = TM / WM / 32, FN = TN / WN / 32;
    constexpr int kStage = SA::kChunks + SB::kChunks;
    static_assert(TM % 64 == 0 && TN % 64 == 0 && SA::KT == kBlock, "whole waves of rows; a block a stage");
    extern __shared__ Chunk stages[];
    unsigned* const words = reinterpret_cast<unsigned*>(stages + RING * kStage);           // [2][TM + TN]
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
    // exponents: 64 rows of the tile at a time, one or two times a wave
    constexpr int kWaves = WM * WN, kPieces = (TM + TN) / 64, kOwn = (kPieces + kWaves - 1) / kWaves;
    const auto scalar = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    Descriptor dw[kOwn];
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
        const int piece = wave + i * kWaves;
        const bool of_a = piece * 64 < TM;
        const int64_t row0 = of_a ? m0 + piece * 64 : n0 + piece * 64 - TM, rows = (of_a ? a.extent : b.extent) - row0;
        const uint64_t at = reinterpret_cast<uint64_t>((of_a ? a.exponents : b.exponents) + row0 * a.padded);
        dw[i] = {scalar(static_cast<int>(at)), scalar(static_cast<int>(at >> 32) & 0xffff), scalar(rows <= 0 ? 0 : static_cast<int>(min<int64_t>(rows, 64)) * a.padded),
                 0x00020000};
    }
    const auto load_words = [&](int group) {                   // (beyond the end: zeros, which nobody uses)
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
            if (wave + i * kWaves < kPieces)
                word_to_lds(dw[i], 4 * group < a.padded ? static_cast<unsigned>(l * a.padded + 4 * group) : kNowhere,
                            scalar(static_cast<int>(reinterpret_cast<uintptr_t>((LdsVoid)(words + (group & 1) * (TM + TN)))) + (wave + i * kWaves) * 256));
    };
    Descriptor da, db;
    const auto load = [&](int s, int i) {
        const Chunk* tile = stages + s % RING * kStage;
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
        const Chunk* tile = stages + s % RING * kStage;
        return f < FM ? Codes32{fragment<Code, true, TM, 8, false>(tile, wm + 32 * f, 2 * h), fragment<Code, true, TM, 8, false>(tile, wm + 32 * f, 2 * h + 1)}
                      : Codes32{fragment<Code, true, TN, 8, true>(tile + SA::kChunks, wn + 32 * (f - FM), 2 * h),
                                fragment<Code, true, TN, 8, true>(tile + SA::kChunks, wn + 32 * (f - FM), 2 * h + 1)};
    };
    const auto slot = [](int h, int j) { return j < FN - 1 ? j : FN - 1 + h; };
    unsigned ea[FM], eb[FN];
    // Float32 results of a block with exponents beyond those of bfloat16: the sums so far wait in scratch memory, where they take no registers.
    volatile float aside[sizeof(T) == 4 ? FN * FM * 16 : 1];
    const auto by_a = [&](int i) { return sizeof(T) == 4 ? held_exponent(static_cast<int>(ea[i])) : static_cast<int>(ea[i]); };
    const auto by_b = [&](int i) { return sizeof(T) == 4 ? held_exponent(static_cast<int>(eb[i])) : static_cast<int>(eb[i]); };
    const auto block_beyond = [&] {
        bool any = false;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < FM; ++i) any |= beyond_bfloat16(static_cast<int>(ea[i]));
#pragma unroll
            for (int i = 0; i < FN; ++i) any |= beyond_bfloat16(static_cast<int>(eb[i]));
            any = __any(any);
        }
        return any;
    };
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
            acc[p / FM][p % FM] = multiply_add8<T, false>(xb[slot(h, p / FM)], by_b(p / FM), xa[h][p % FM], by_a(p % FM), acc[p / FM][p % FM]);
            // (keeps the product here: it would be moved behind all loads and reads of the stage, and spill)
            if constexpr (kProducts > 8) asm volatile("" : "+a"(acc[p / FM][p % FM]));
            else asm volatile("" : "+v"(acc[p / FM][p % FM]));
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    if (steps > 0) {
        load_words(first / 4);
#pragma unroll
        for (int s = 0; s < RING - (RING == 2); ++s)
#pragma unroll
            for (int i = 0; i < kLoads; ++i) load(s, i);
        settle<RING == 2 ? 0 : (RING - 1) * kLoads>();         // stage 0 and the words have landed
#pragma unroll
        for (int i = 0; i < FM; ++i) xa[0][i] = take(0, 0, i);
#pragma unroll
        for (int i = 0; i < FN; ++i) xb[slot(0, i)] = take(0, 0, FM + i);
        if constexpr (RING == 2) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) load(1, i);
        }
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
        const bool beyond = block_beyond();
        if (beyond) {
            each<FN * FM * 16>([&](int i) {
                aside[i] = acc[i / 16 / FM][i / 16 % FM][i % 16];
                acc[i / 16 / FM][i / 16 % FM][i % 16] = 0.0f;
            });
        }
        step(0, s, -1);
        // stage s + 1 has landed, and the rest of this one is in registers. (Words are older than the loads of the three stages behind them by the
        // time that they are used.)
        static_assert(RING <= 4, "words land in time");
        settle<(RING - 2) * kLoads>();
        step(1, s + 1, s + RING);
        if (beyond) {
            each<FN * FM * 16>([&](int i) {
                const int f = i / 16 / FM, g = i / 16 % FM, of_b = static_cast<int>(eb[f] & 255) - by_b(f), of_a = static_cast<int>(ea[g] & 255) - by_a(g);
                acc[f][g][i % 16] = aside[i] + ldexpf(acc[f][g][i % 16], of_a + __shfl(of_b, first_row(acc[f][g], i % 16)));
            });
        }
#pragma unroll
        for (int i = 0; i < FM; ++i) ea[i] >>= 8;
#pragma unroll
        for (int i = 0; i < FN; ++i) eb[i] >>= 8;
    }
    settle<0>();                                               // every wave's loads have landed and its fragments are read: the LDS is free
    static_assert(WM * WN * 256 * FN <= RING * kStage, "each wave turns its sums in a part of the stages");
    store_blocks<T, FN, FM>(tail, acc, m0 + wm, n0 + wn, part, stages + wave * 256 * FN);
}

// ---- few rows --------------------------------------------------------------------------------------------------------
// y for at most 16 * MT rows: the weight's codes are all there is to read, once. A workgroup takes 16 columns n and its waves share k. A wave
// brings `ahead` blocks of its 16 rows of the weight to LDS at a time (fragments read straight from memory would touch four times as many cache
// lines per load), and reads its fragments there. CODED: x is codes, which come the same way; else values, quantized on the way in registers: the
// four lanes that hold a row's share of a block agree on its exponent. That saves a launch, and the few rows come from the caches.
// Bound by the launch and one way to memory and back: one row of 1024 -> 4096 bfloat16 5.2 us (with two launches the call took 11.4 us, 8.4 this way).
template <class T>
__device__ __forceinline__ void quantize_share(const T* p, int64_t left, Codes32& codes, int& exponent) {
    float v[32];
    constexpr int V = Vec<T>::kLen;
#pragma unroll
    for (int i = 0; i < 32; i += V) {
        T part[V];
        load_run<T, V>(p + i, part, left - i);
#pragma unroll
        for (int j = 0; j < V; ++j) v[i + j] = static_cast<float>(part[j]);
    }
    float most = largest(v);
    most = fmaxf(most, partner<16>(most));
    most = fmaxf(most, partner<32>(most));
    exponent = block_exponent(most);
    const Codes<32> c = to_codes(v, exponent);
    codes = __builtin_bit_cast(Codes32, c);
}

template <class T, int MT, bool CODED>
__global__ void __launch_bounds__(512)
few_rows_float8_kernel(Coded a, const T* x, int64_t ld_x, int64_t columns, Coded b, Tail<T> tail, int ahead) {
    extern __shared__ Chunk blocks[];
    const int l = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), waves = blockDim.x / 64;
    const int64_t n0 = blockIdx.x * 16ll;
    const int count = a.blocks, part = (count + waves - 1) / waves, last = min(count, (wave + 1) * part);
    constexpr int kRows = 16 * (CODED ? MT + 1 : 1);           // rows of the weight, then of x
    Chunk* const mine = blocks + wave * kRows * 8 * ahead;
    const unsigned to = static_cast<unsigned>(reinterpret_cast<uintptr_t>((LdsVoid)mine));
    const int ld = count * kBlock, rows_w = static_cast<int>(min<int64_t>(16, b.extent - n0)), rows_x = static_cast<int>(a.extent);
    const auto describe = [](const uint8_t* p, int64_t size) {
        const uint64_t at = reinterpret_cast<uint64_t>(p);
        return Descriptor{__builtin_amdgcn_readfirstlane(static_cast<int>(at)), __builtin_amdgcn_readfirstlane(static_cast<int>(at >> 32) & 0xffff),
                          __builtin_amdgcn_readfirstlane(static_cast<int>(size)), 0x00020000};
    };
    const Descriptor dw = describe(b.codes + n0 * ld, static_cast<int64_t>(rows_w) * ld), dx = describe(a.codes, CODED ? static_cast<int64_t>(rows_x) * ld : 0);
    const uint8_t* w_exponents = b.exponents + min(n0 + l % 16, b.extent - 1) * b.padded;
    Acc4 acc[MT] = {};
    for (int s = wave * part; s < last; s += ahead) {
        // chunk c of row r lies at c ^ r, whose low bits keep neighbouring rows in different banks
        const int chunks = 8 * ahead, mask = chunks - 1;
        for (int i = 0; i < kRows * ahead / 8; ++i) {
            const int q = i * 64 + l, r = q / chunks, c = (q & mask) ^ (r & mask), k = s * kBlock + c * 16, row = r < 16 ? r : r - 16;
            const bool inside = k < ld && row < (r < 16 ? rows_w : rows_x);
            load_to_lds(i * 64 / chunks < 16 ? dw : dx, inside ? static_cast<unsigned>(row * ld + k) : kNowhere, __builtin_amdgcn_readfirstlane(to + i * 1024));
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // (a wave's blocks are its own)
        for (int j = 0; j < ahead && s + j < last; ++j) {
            const int r = l % 16, c = 8 * j + l / 16 * 2;
            const auto from_lds = [&](int row) { return Codes32{mine[row * chunks + (c ^ (row & mask))], mine[row * chunks + ((c + 1) ^ (row & mask))]}; };
            const Codes32 w = from_lds(r);
            const int ew = w_exponents[s + j];
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                Codes32 v;
                int e;
                if constexpr (CODED) {
                    v = from_lds(16 + 16 * i + r);
                    e = a.exponents[min(16 * i + r, rows_x - 1) * a.padded + s + j];
                } else {
                    const int64_t k = static_cast<int64_t>(s + j) * kBlock + l / 16 * 32;
                    // (rows beyond the end repeat the last one: nobody stores their sums)
                    quantize_share(x + min(16 * i + r, rows_x - 1) * ld_x + k, columns - k, v, e);
                }
                with_exponents<T>(beyond_bfloat16(e) || beyond_bfloat16(ew), [&](auto far) { acc[i] = multiply_add8<T, decltype(far)::value>(w, ew, v, e, acc[i]); });
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");     // read before the next blocks overwrite them
    }
    __syncthreads();
    Acc4* sums = reinterpret_cast<Acc4*>(blocks);
#pragma unroll
    for (int i = 0; i < MT; ++i) sums[(wave * MT + i) * 64 + l] = acc[i];
    __syncthreads();
    for (int i = wave; i < MT; i += waves) {
        float z[4] = {};
        for (int w = 0; w < waves; ++w) {
            const Acc4 v = sums[(w * MT + i) * 64 + l];
#pragma unroll
            for (int r = 0; r < 4; ++r) z[r] += v[r];
        }
        apply_tail<T, 4>(tail, z, 16 * i + l % 16, n0 + 4 * (l / 16));
    }
}

// ---- few channels ----------------------------------------------------------------------------------------------------
// y of many rows through a weight of at most KB blocks a row that LDS holds whole. A wave takes 32 rows at a time with all their columns: its
// lanes read the row's values (or, CODED, its codes) once, two lanes a row, and quantize them in registers; the codes never go through memory.
// Then 32 columns at a time: products, epilogue. Workgroups of eight waves go round over the rows. WHOLE: rows of values end with a block.
// Bound by memory: 131072 x 128 -> 32 bfloat16 with relu 11.4 to 11.9 us repeated alone, 3.6 TB/s of values in and results out, 12.4 to 13.2 among passes on other
// inputs (quantized first and through tiles 24.2). Float32 22.8 us.
constexpr int kNarrowBlocks = 4, kNarrowWaves = 8;         // (a row's exponents are one word)
constexpr size_t kNarrowWeight = 64 * 1024;
constexpr size_t narrow_float8_lds(int64_t columns, int blocks) { return static_cast<size_t>((columns + 31) / 32 * 32) * (blocks * kBlock + 4) + kNarrowWaves * 4096; }

template <class T, int KB, bool CODED, bool WHOLE>
__global__ void __launch_bounds__(kNarrowWaves * 64, KB == 1 && WHOLE && sizeof(T) == 2 ? 4 : 2)
narrow_float8_kernel(Coded a, const T* x, int64_t ld_x, int64_t columns, Coded b, Tail<T> tail) {
    typedef TileShape<Code, true, 32, 8> Tile;
    extern __shared__ Chunk lds[];
    const int l = threadIdx.x % 64, wave = threadIdx.x / 64, rows_w = static_cast<int>(b.extent + 31) / 32 * 32;
    Chunk* const turn = lds + wave * 256;                      // where a wave turns its sums
    Chunk* const weight = lds + kNarrowWaves * 256;            // [KB][rows_w][8]
    unsigned* const words = reinterpret_cast<unsigned*>(weight + KB * rows_w * 8);
    for (int i = threadIdx.x; i < KB * rows_w * 8; i += kNarrowWaves * 64) {
        const int row = i / (KB * 8), c = i % (KB * 8);
        const Chunk v = row < b.extent ? *reinterpret_cast<const Chunk*>(b.codes + (row * KB * 8 + c) * 16ll) : Chunk{0, 0, 0, 0};
        weight[c / 8 * rows_w * 8 + Tile::place<true>(row, c % 8)] = v;
    }
    for (int i = threadIdx.x; i < rows_w; i += kNarrowWaves * 64) words[i] = i < b.extent ? *reinterpret_cast<const unsigned*>(b.exponents + i * 4ll) : 0x7f7f7f7fu;
    __syncthreads();
    bool weight_beyond = false;
    if constexpr (sizeof(T) == 4) {
        for (int i = l; i < rows_w; i += 64) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) weight_beyond |= beyond_bfloat16(static_cast<int>(words[i] >> 8 * kb));
        }
    }
    for (int64_t m0 = (blockIdx.x * static_cast<int64_t>(kNarrowWaves) + wave) * 32; m0 < a.extent; m0 += gridDim.x * static_cast<int64_t>(kNarrowWaves * 32)) {
        // (rows beyond the end repeat the last one: nobody stores their sums)
        const int64_t m = min(m0 + l % 32, a.extent - 1);
        Codes32 codes[KB][2];
        int ea[KB];
        if constexpr (CODED) {
            const unsigned word = *reinterpret_cast<const unsigned*>(a.exponents + m * 4);
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                ea[kb] = static_cast<int>(word >> 8 * kb);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const Chunk* p = reinterpret_cast<const Chunk*>(a.codes + m * (KB * kBlock) + kb * kBlock) + 4 * h + l / 32;
                    codes[kb][h] = {p[0], p[2]};
                }
            }
        } else {
            const T* p = x + m * ld_x;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                // chunks l / 32 and l / 32 + 2 of each half, as the weight's fragments have them
                float v[64];
                constexpr int V = Vec<T>::kLen;
                typename Vec<T>::Type raw[64 / V] = {};
                const auto k_of = [&](int i) { return kb * kBlock + i * V / 16 * 32 + l / 32 * 16 + i * V % 16; };
                if constexpr (WHOLE) {
#pragma unroll
                    for (int i = 0; i < 64 / V; ++i) raw[i] = *reinterpret_cast<const typename Vec<T>::Type*>(p + k_of(i));
                } else {                                       // (rows hold a vector at least)
                    Chunk part[64 / V];
#pragma unroll
                    for (int i = 0; i < 64 / V; ++i) part[i] = request_chunk(p + k_of(i), static_cast<int>(columns) - k_of(i), x);
#pragma unroll
                    for (int i = 0; i < 64 / V; ++i) {
                        settle_chunk<T>(part[i], static_cast<int>(columns) - k_of(i));
                        raw[i] = __builtin_bit_cast(typename Vec<T>::Type, part[i]);
                    }
                }
#pragma unroll
                for (int i = 0; i < 64; ++i) v[i] = static_cast<float>(raw[i / V][i % V]);
                float most = largest(v);
                most = fmaxf(most, partner<32>(most));
                ea[kb] = block_exponent(most);
                const Codes<64> c = to_codes(v, ea[kb]);
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    codes[kb][h] = {Chunk{c[8 * h], c[8 * h + 1], c[8 * h + 2], c[8 * h + 3]}, Chunk{c[8 * h + 4], c[8 * h + 5], c[8 * h + 6], c[8 * h + 7]}};
            }
        }
        bool beyond = weight_beyond;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) beyond |= beyond_bfloat16(ea[kb]);
        }
        const auto columns_from = [&](auto far, int n0) {
            Acc16 acc[1][1] = {};
            const unsigned word = words[n0 + column_of(l % 32)];
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                const Chunk* tile = weight + kb * rows_w * 8;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const Codes32 w = {fragment<Code, true, 32, 8, true>(tile, n0, 2 * h), fragment<Code, true, 32, 8, true>(tile, n0, 2 * h + 1)};
                    acc[0][0] = multiply_add8<T, decltype(far)::value>(w, static_cast<int>(word >> 8 * kb), codes[kb][h], ea[kb], acc[0][0]);
                }
            }
            store_blocks<T, 1, 1>(tail, acc, m0, n0, 0, turn);
        };
        if constexpr (sizeof(T) == 2) {
            for (int n0 = 0; n0 < b.extent; n0 += 32) columns_from(std::false_type(), n0);
        } else {
            with_exponents<T>(beyond, [&](auto far) {
                for (int n0 = 0; n0 < b.extent; n0 += 32) columns_from(far, n0);
            });
        }
    }
}

}  // namespace

}  // namespace boxconv
