// The pointwise product for operands whose rows are whole aligned 16-byte chunks: tiles come into LDS directly from memory.
#pragma once

#include "linear_tile.hpp"

namespace boxconv {

namespace {

// 16 bytes per lane from `offset` bytes into a descriptor's memory to LDS at `to` + 16 * lane; offsets at or beyond the
// descriptor's size give zeros. In assembly because the compiler waits for all such loads in front of every transposed LDS
// read; it writes no register, and settle() does the waiting. (One wait state between the write of M0 and its use.)
constexpr unsigned kNowhere = 0xfffffff0u;                             // beyond every size
typedef __attribute__((address_space(3))) const void* LdsVoid;
typedef int Descriptor __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void load_to_lds(Descriptor d, unsigned offset, unsigned to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(offset), "s"(d) : "m0");
}

// One operand's tile as the DMA fills it: where each of a thread's chunks comes from.
template <class T, bool K_MAJOR, int X, int THREADS, bool PERM>
struct Feed {
    typedef TileShape<T, K_MAJOR, X, 8> Shape;
    static constexpr int N = Shape::kChunks / THREADS;
    static_assert(!K_MAJOR || THREADS % 256 == 0, "a thread's chunks of a K-major tile all have the same k");
    unsigned off[N];           // bytes from the tile's corner in memory; kNowhere for rows beyond the operand
    int k;                     // K-major: first k of the thread's chunks, from the tile's
    const char* base;          // the corner, of the next tile to fetch
    int64_t size;              // bytes from there to the operand's end
    int64_t step;              // bytes to the next tile

    __device__ __forceinline__ void start(const Operand<T>& o, int64_t i0, int64_t k0) {
        const int64_t ld = o.ld * static_cast<int64_t>(sizeof(T));
#pragma unroll
        for (int s = 0; s < N; ++s) {
            // chunk q of the tile holds what `place` puts there (an exclusive-or of the column: its own inverse)
            const int q = threadIdx.x + s * THREADS, r = q / Shape::kRowChunks, c = Shape::template place<PERM>(r, q % Shape::kRowChunks) % Shape::kRowChunks;
            const bool inside = K_MAJOR ? i0 + r < o.extent : i0 + c * Shape::V < o.extent;
            off[s] = inside ? static_cast<unsigned>(r * ld + c * 16) : kNowhere;
            k = c * Shape::V;
        }
        const int64_t corner = K_MAJOR ? i0 * ld + k0 * static_cast<int64_t>(sizeof(T)) : k0 * ld + i0 * static_cast<int64_t>(sizeof(T));
        const int64_t bytes = ((K_MAJOR ? o.extent : o.depth) - 1) * ld + (K_MAJOR ? o.depth : o.extent) * static_cast<int64_t>(sizeof(T));
        base = reinterpret_cast<const char*>(o.p) + corner;
        size = bytes - corner;
        step = K_MAJOR ? 128 : Shape::KT * ld;
    }
    // The descriptor of the next tile.
    __device__ __forceinline__ Descriptor next() {
        const unsigned bytes = size <= 0 ? 0u : size < 0xffffff00ll ? static_cast<unsigned>(size) : 0xffffff00u;
        const uint64_t at = reinterpret_cast<uint64_t>(base);
        base += step;
        size -= step;
        return {static_cast<int>(at), static_cast<int>(at >> 32) & 0xffff, static_cast<int>(bytes), 0x00020000};
    }
    // The thread's chunk s of it, with its workgroup's others, into `tile`. k_left: values of k from the tile's corner to the
    // end of the sum, none where it is <= 0: a K-major operand's chunks beyond it would be the next row's. (Rows of k beyond
    // the other kind's end are beyond its descriptor.)
    __device__ __forceinline__ void fetch(Descriptor d, int s, const Chunk* tile, int k_left) const {
        const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
        const unsigned to = static_cast<unsigned>(reinterpret_cast<uintptr_t>((LdsVoid)(tile + s * THREADS))) + wave * 1024;
        load_to_lds(d, !K_MAJOR || k < k_left ? off[s] : kNowhere, to);
    }
};

// Tile and part of k of this workgroup: neighbours share an XCD's L2 (the hardware deals workgroups to the eight XCDs in turn), the
// tiles of one part among them, which read the same rows (200000 rows, 256 x 256 weight gradient in parts of four tiles: 66 us with the tiles on four XCDs, 53 on one), and
// walk down 8 tiles of m before the next n.
__device__ __forceinline__ void tile_of(unsigned tiles_m, unsigned tiles_n, unsigned& tm, unsigned& tn, unsigned& part) {
    const unsigned tiles = tiles_m * tiles_n, total = tiles * gridDim.y, whole = total / 8 * 8;
    unsigned id = blockIdx.y * tiles + blockIdx.x;
    if (id < whole) id = id % 8 * (whole / 8) + id / 8;
    part = id / tiles;
    id -= part * tiles;
    const unsigned group = id / (8 * tiles_n), first = group * 8, high = min(8u, tiles_m - first), rest = id - group * 8 * tiles_n;
    tm = first + rest % high;
    tn = rest / high;
}

constexpr int kRing = 2;           // stages of LDS

// At most N of this wave's loads may still be on their way and none of its LDS reads; then wait for every wave to get here.
template <int N>
__device__ __forceinline__ void settle() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory"); }

// TM x TN tile by WM x WN waves, each with (TM/WM) x (TN/WN). Two stages of 128 bytes of k. The barrier of a stage stands in front
// of its last k step, whose fragments are in registers by then: from there on its LDS takes the stage after next, whose loads are
// issued one at a time between the products of two k steps (eight waves that issue theirs all at once keep the memory pipe,
// and with it themselves, busy for half a stage), and the next stage's first fragments are read between the last products.
// Bound by the matrix instructions and the power they draw. Each repeated alone, bfloat16: 8192 x 2048 -> 4096 119 us (1.16 PFLOP/s), 133 with gelu and
// bias, where a library product takes 98 to 112; 8192 x 4096 -> 2048 109 us, dx 118, dW 136 against 90 to 100, 113 to 129 and 128 to 147. One after
// the other in a training step the clock is lower: y with silu, a residual and a kept slope 146 us, dx 133, dW 164. (On zeros everything is
// 20 % faster.) No better: four stages of 64 bytes of k, waves of 128 x 128 (they spill), wave priorities.
template <class T, bool A_K, bool B_K, int TM, int TN, int WM, int WN>
__global__ void __launch_bounds__(WM * WN * 64)
product_wide_kernel(Operand<T> a, Operand<T> b, Tail<T> tail, int64_t k_part, unsigned tiles_m, unsigned tiles_n) {
    typedef TileShape<T, A_K, TM, 8> SA;
    typedef TileShape<T, B_K, TN, 8> SB;
    constexpr int THREADS = WM * WN * 64, FM = TM / WM / 32, FN = TN / WN / 32;
    constexpr int kStage = SA::kChunks + SB::kChunks;
    extern __shared__ Chunk stages[];
    unsigned tm, tn, part;
    tile_of(tiles_m, tiles_n, tm, tn, part);
    const int64_t m0 = static_cast<int64_t>(tm) * TM, n0 = static_cast<int64_t>(tn) * TN;
    const int64_t k_begin = part * k_part, k_end = min(a.depth, k_begin + k_part);
    const int wave = threadIdx.x / 64, wm = wave / WN * (TM / WM), wn = wave % WN * (TN / WN);
    Acc16 acc[FN][FM] = {};
    typedef Feed<T, A_K, TM, THREADS, false> FeedA;
    typedef Feed<T, B_K, TN, THREADS, true> FeedB;
    FeedA fa;
    FeedB fb;
    fa.start(a, m0, k_begin);
    fb.start(b, n0, k_begin);
    const int depth = static_cast<int>(k_end - k_begin), steps = (depth + SA::KT - 1) / SA::KT;
    Descriptor da, db;
    // piece i of the loads of stage s of the sum (beyond its end: zeros, which nobody uses)
    const auto load = [&](int s, int i) {
        const Chunk* tile = stages + s % kRing * kStage;
        const int k_left = depth - s * SA::KT;
        if (i == 0) da = fa.next();
        if (i == FeedA::N) db = fb.next();
        if (i < FeedA::N) fa.fetch(da, i, tile, k_left);
        else fb.fetch(db, i - FeedA::N, tile + SA::kChunks, k_left);
    };
    Chunk xa[2][FM], xb[2][FN];
    // piece i of the fragments of k step ks of stage s
    const auto read = [&](int s, int ks, int i) {
        const Chunk* tile = stages + s % kRing * kStage;
        if (i < FM) xa[ks & 1][i] = fragment<T, A_K, TM, 8, false>(tile, wm + 32 * i, ks);
        else xb[ks & 1][i - FM] = fragment<T, B_K, TN, 8, true>(tile + SA::kChunks, wn + 32 * (i - FM), ks);
    };
    constexpr int kLoads = FeedA::N + FeedB::N, kReads = FM + FN, kProducts = FM * FN;     // of a thread: per stage, k step, k step
    // k step ks: its products, and between them loads [first, last) of stage `to` and the reads of the k step after it, of stage `from`
    const auto step = [&](int ks, int from, int to, int first, int last) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int p = 0; p < kProducts; ++p) {
#pragma unroll
            for (int i = p * kReads / kProducts; i < (p + 1) * kReads / kProducts; ++i) read(from, (ks + 1) % 4, i);
#pragma unroll
            for (int i = p * (last - first) / kProducts; i < (p + 1) * (last - first) / kProducts; ++i) load(to, first + i);
            acc[p / FM][p % FM] = multiply_add<T>(xb[ks & 1][p / FM], xa[ks & 1][p % FM], acc[p / FM][p % FM]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    static_assert(SA::kSteps == 4, "four k steps in a stage");
    constexpr int kHalf = (kLoads + 1) / 2;
    if (steps > 0) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) load(0, i);
        settle<0>();
#pragma unroll
        for (int i = 0; i < kReads; ++i) read(0, 0, i);
#pragma unroll
        for (int i = 0; i < kHalf; ++i) load(1, i);
    }
    for (int s = 0; s < steps; ++s) {
        step(0, s, s + 1, kHalf, kLoads);
        step(1, s, 0, 0, 0);
        step(2, s, 0, 0, 0);
        settle<0>();                                           // stage s + 1 has landed, and the rest of this one is in registers
        step(3, s + 1, s + 2, 0, kHalf);
    }
    settle<0>();                                               // every wave's loads have landed and its fragments are read: the LDS is free
    static_assert(WM * WN * 256 * FN <= kRing * kStage, "each wave turns its sums in a part of the stages");
    store_blocks<T, FN, FM>(tail, acc, m0 + wm, n0 + wn, part, stages + wave * 256 * FN);
}

}  // namespace

}  // namespace boxconv
