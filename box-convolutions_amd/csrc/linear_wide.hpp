// The pointwise product for operands whose rows are whole aligned 16-byte chunks: tiles come into LDS directly from memory.
#pragma once

#include "linear_tile.hpp"

namespace boxconv {

namespace {

// Loads of up to 64 lanes x 16 bytes from a descriptor's memory into LDS at `to` + 16 * lane. Offsets at or beyond the
// descriptor's size give zeros; kNowhere is beyond every size.
constexpr unsigned kNowhere = 0xfffffff0u;
typedef __attribute__((address_space(3))) void LdsVoid;

// One operand's tile as the DMA fills it: where each of a thread's chunks comes from.
template <class T, bool K_MAJOR, int X, int THREADS, bool PERM>
struct Feed {
    typedef TileShape<T, K_MAJOR, X> Shape;
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
    // The next tile into `tile`. k_left: values of k from its corner to the end of the sum, none where it is <= 0: a K-major
    // operand's chunks beyond it would be the next row's. (Rows of k beyond the other kind's end are beyond its descriptor.)
    __device__ __forceinline__ void fetch(Chunk* tile, int k_left) {
        const unsigned bytes = size <= 0 ? 0u : size < 0xffffff00ll ? static_cast<unsigned>(size) : 0xffffff00u;
        const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, static_cast<int>(bytes), 0x00020000);
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
        const bool inside = !K_MAJOR || k < k_left;
#pragma unroll
        for (int s = 0; s < N; ++s)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (LdsVoid*)(tile + s * THREADS + wave * 64), 16, static_cast<int>(inside ? off[s] : kNowhere), 0, 0, 0);
        base += step;
        size -= step;
    }
};

// Tile m0, n0 of workgroup `id`: neighbours in id share an XCD's L2 (the hardware deals workgroups to the eight XCDs in
// turn) and walk down 8 tiles of m before the next n.
__device__ __forceinline__ void tile_of(unsigned id, unsigned tiles_m, unsigned tiles_n, unsigned& tm, unsigned& tn) {
    const unsigned total = tiles_m * tiles_n, whole = total / 8 * 8;
    if (id < whole) id = id % 8 * (whole / 8) + id / 8;
    const unsigned group = id / (8 * tiles_n), first = group * 8, high = min(8u, tiles_m - first), rest = id - group * 8 * tiles_n;
    tm = first + rest % high;
    tn = rest / high;
}

// TM x TN tile by WM x WN waves, each with (TM/WM) x (TN/WN). Two stages of LDS: while one is multiplied the other fills.
template <class T, bool A_K, bool B_K, int TM, int TN, int WM, int WN>
__global__ void __launch_bounds__(WM * WN * 64)
product_wide_kernel(Operand<T> a, Operand<T> b, Tail<T> tail, int64_t k_part, unsigned tiles_m, unsigned tiles_n) {
    typedef TileShape<T, A_K, TM> SA;
    typedef TileShape<T, B_K, TN> SB;
    constexpr int THREADS = WM * WN * 64, FM = TM / WM / 32, FN = TN / WN / 32;
    constexpr int kStage = SA::kChunks + SB::kChunks;
    extern __shared__ Chunk stages[];
    unsigned tm, tn;
    tile_of(blockIdx.x, tiles_m, tiles_n, tm, tn);
    const int64_t m0 = static_cast<int64_t>(tm) * TM, n0 = static_cast<int64_t>(tn) * TN;
    const int64_t k_begin = blockIdx.y * k_part, k_end = min(a.depth, k_begin + k_part);
    const int wave = threadIdx.x / 64, wm = wave / WN * (TM / WM), wn = wave % WN * (TN / WN);
    Acc16 acc[FN][FM] = {};
    Feed<T, A_K, TM, THREADS, false> fa;
    Feed<T, B_K, TN, THREADS, true> fb;
    fa.start(a, m0, k_begin);
    fb.start(b, n0, k_begin);
    int left = static_cast<int>(k_end - k_begin);              // of k, from the next tile to fetch on
    const int steps = (left + SA::KT - 1) / SA::KT;
    const auto fetch = [&](int stage) {
        fa.fetch(stages + stage * kStage, left);
        fb.fetch(stages + stage * kStage + SA::kChunks, left);
        left -= SA::KT;
    };
    Chunk xa[2][FM], xb[2][FN];
    const auto read = [&](const Chunk* tile, int ks) {
#pragma unroll
        for (int j = 0; j < FM; ++j) xa[ks & 1][j] = fragment<T, A_K, TM, false>(tile, wm + 32 * j, ks);
#pragma unroll
        for (int i = 0; i < FN; ++i) xb[ks & 1][i] = fragment<T, B_K, TN, true>(tile + SA::kChunks, wn + 32 * i, ks);
    };
    const auto multiply = [&](int ks) {
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int j = 0; j < FM; ++j) acc[i][j] = multiply_add<T>(xb[ks & 1][i], xa[ks & 1][j], acc[i][j]);
    };
    // the fragments of the next k step are requested one at a time between the products of this one
    const auto interleave = [] {
        constexpr int kReads = FM * (A_K ? 1 : sizeof(T) == 2 ? 2 : 4) + FN * (B_K ? 1 : sizeof(T) == 2 ? 2 : 4);
        constexpr int kProducts = FM * FN * (sizeof(T) == 2 ? 1 : 4), kEach = (kReads + kProducts - 1) / kProducts;
#pragma unroll
        for (int i = 0; i < kProducts; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, kEach, 0);     // LDS reads
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);         // matrix instructions
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    // this wave's share of the outstanding stage has landed and its own reads are done; then everybody's
    const auto settle = [] { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    if (steps > 0) {
        fetch(0);
        settle();
        fetch(1);
        read(stages, 0);
    }
    for (int s = 0; s < steps; ++s) {
        const Chunk* now = stages + (s & 1) * kStage;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < 3; ++ks) {
            read(now, ks + 1);
            multiply(ks);
            interleave();
        }
        // the last fragments of this stage are on their way: once they are here, its LDS is free for the stage after next, and
        // the next stage's first fragments can be requested before the last products. (Behind the last stage this fetches
        // and reads what nobody uses: zeros, or the stage before.)
        settle();
        fetch(s & 1);
        read(stages + (~s & 1) * kStage, 0);
        multiply(3);
        interleave();
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");           // nothing may still be on its way into this workgroup's LDS when it ends
    const int l = threadIdx.x % 64;
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            const int64_t m = m0 + wm + 32 * j + l % 32, n = n0 + wn + 32 * i + 16 * (l / 32);
            float z[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) z[r] = acc[i][j][r];
            if (tail.partial != nullptr) {
                if (m < tail.rows && n < tail.cols)
                    store_run<float, 16>(tail.partial + (blockIdx.y * tail.rows + m) * tail.cols + n, z, tail.cols - n);
            } else {
                apply_tail<T, 16>(tail, z, m, n);
            }
        }
}

}  // namespace

}  // namespace boxconv
