// Backward of the pointwise product through few channels: one pass over x and grad_output.
//
// With K and N of a few dozen or hundred (a 1 x 1 convolution) both gradients are bound by memory, and computed one after the
// other they read dz and x twice and write dz once. Here a workgroup of eight waves keeps the weight in LDS and walks over tiles of
// TM rows: dz = dy * act' goes from registers to LDS, x straight to LDS, dx = dz W leaves for memory, and the workgroup's share
// of dW = dz^T x and of the column sums of dz stays in registers until its last tile. The shares are added by another
// launch, in a fixed order.
//
// LDS rows are padded instead of permuted, since K and N are known at run time only: a pitch of 64 bytes times an odd number for
// transposed reads in 16-bit types (four rows of 64 bytes side by side in the 256 bytes of a bank cycle), 32 times an odd number
// for reads of single floats (rows k and k + 4 side by side), 16 times an odd number for 16-byte reads of one chunk of many rows.
#pragma once

#include "linear_wide.hpp"

namespace boxconv {

namespace {

template <class T>
struct NarrowArgs {
    const T *x, *weight, *dy;
    const void* kept;
    int64_t ld_x, rows;
    T *dx, *dresidual;
    float *dweight, *dbias;      // [workgroups][N][K], [workgroups][N]; dweight and dbias may be null
    int N, K, activation, tiles;
};

// Pitches in chunks and sizes in bytes.
struct NarrowLds {
    int px, pa, pb;              // rows of x and the weight; rows of dz for 16-byte reads; for transposed ones
    int x_bytes, a_bytes, b_bytes, w_bytes;
    __host__ __device__ constexpr int total() const { return 2 * (x_bytes + a_bytes + b_bytes) + w_bytes + 128; }   // (a fragment may reach 96 bytes past the last row)
};
template <class T>
__host__ __device__ constexpr NarrowLds narrow_lds(int N, int K, int TM) {
    constexpr int V = Vec<T>::kLen;
    NarrowLds s = {};
    const int cx = K / V, cn = (N / V + 1) / 2 * 2;                       // (whole k steps of n)
    if (sizeof(T) == 2) {
        s.px = cx + (12 - cx % 8) % 8;
        s.pb = cn + (12 - cn % 8) % 8;
    } else {
        s.px = cx + (6 - cx % 4) % 4;
        s.pb = 0;                                                         // (float: both kinds of reads from the one copy)
    }
    s.pa = cn + 1;
    s.x_bytes = (TM * s.px + 63) / 64 * 1024;
    s.a_bytes = TM * s.pa * 16;
    s.b_bytes = TM * s.pb * 16;
    s.w_bytes = (cn * V * s.px + 63) / 64 * 1024;
    return s;
}
// Rows of column sums that the workgroup's threads hold at the end, N floats each: those of one pass over a tile, as far as the tile reaches.
template <class T>
__host__ __device__ constexpr int narrow_sum_rows(int N, int TM) {
    const int per_pass = 512 / (N / Vec<T>::kLen);
    return per_pass < TM ? per_pass : TM;
}
// The column sums take the place of the tiles and have to fit there, for every K and N the kernel may be asked for.
template <class T>
constexpr bool sums_fit() {
    for (int N = Vec<T>::kLen; N <= 128; N += Vec<T>::kLen)
        for (int K = Vec<T>::kLen; K <= 1024; K += Vec<T>::kLen)
            for (int TM = 32; TM <= 64; TM *= 2)
                if (narrow_sum_rows<T>(N, TM) * N * 4 > narrow_lds<T>(N, K, TM).total()) return false;
    return true;
}
static_assert(sums_fit<BOXCONV_INST_T>(), "column sums beyond the LDS of the tiles");

// A transposed fragment (32 columns from `i` on, k step ks of the rows) of a tile of `pitch` chunks per row.
template <class T, bool PERM>
__device__ __forceinline__ Chunk transposed(const char* tile, int pitch, int i, int ks) {
    const int l = threadIdx.x % 64;
    if constexpr (sizeof(T) == 2) {
        typedef short Four __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) Four* LdsPtr;
        const int s = l % 16, q = l / 16, four = 4 * (q & 1) + s % 4;
        const int col = i + (PERM ? 16 * (four & 1) + 4 * (four >> 1) : 4 * four);
        const int k = 16 * ks + 8 * (q >> 1) + s / 4;
        const Four lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(tile + k * pitch * 16 + col * 2));
        const Four hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(tile + (k + 4) * pitch * 16 + col * 2));
        typedef short Eight __attribute__((ext_vector_type(8)));
        return __builtin_bit_cast(Chunk, Eight(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7)));
    } else {
        typedef float Four __attribute__((ext_vector_type(4)));
        const int col = i + (PERM ? column_of(l % 32) : l % 32), k = 8 * ks + 4 * (l / 32);
        Four v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const float*>(tile + (k + j) * pitch * 16 + col * 4);
        return __builtin_bit_cast(Chunk, v);
    }
}

// BLOCKS: 32 x 32 blocks of dW that a wave sums.
// 131072 rows, 128 -> 32 bfloat16 21 us (84 MB, 3.9 TB/s), 64 -> 64 float16 20 us; 65536 rows, 256 -> 64 float 71 us, of which the matrix
// instructions take 33: one workgroup of 512 threads fills a compute unit, and its phases (loads, dz to LDS, products, stores) follow each
// other. Without dx it takes 42 us, without dW 56, without either 24. Fragments of the weight held in registers, or of x used twice, gained
// nothing in float and cost 7 us in bfloat16.
template <class T, int TM, int BLOCKS>
__global__ void __launch_bounds__(512)
narrow_grad_kernel(NarrowArgs<T> a) {
    typedef typename SlopeOf<T>::Type S;
    constexpr int V = Vec<T>::kLen, STEP = 2 * V;                          // values of the summed index per k step
    extern __shared__ Chunk lds_chunks[];
    char* lds = reinterpret_cast<char*>(lds_chunks);
    const NarrowLds s = narrow_lds<T>(a.N, a.K, TM);
    char *xs = lds, *das = xs + 2 * s.x_bytes, *dbs = das + 2 * s.a_bytes, *ws = dbs + 2 * s.b_bytes;
    const int t = threadIdx.x, l = t % 64, wave = __builtin_amdgcn_readfirstlane(t / 64);
    const int chunks_k = a.K / V, chunks_n = a.N / V, blocks_k = (a.K + 31) / 32, blocks_n = (a.N + 31) / 32;

    // the weight, and with it zeros in its padding and its rows beyond N
    const unsigned lds_base = static_cast<unsigned>(reinterpret_cast<uintptr_t>((LdsVoid)lds_chunks));
    const int down = 512 / s.px, across = 512 % s.px;                      // from a thread's chunk of a padded tile to its next one
    const auto fetch = [&](const T* from, int64_t ld, int64_t rows, int tile_rows, unsigned to) {
        const int64_t step = ld * static_cast<int64_t>(sizeof(T)), size = rows <= 0 ? 0 : (rows - 1) * step + static_cast<int64_t>(a.K) * static_cast<int64_t>(sizeof(T));
        const uint64_t at = reinterpret_cast<uint64_t>(from);
        const Descriptor desc = {static_cast<int>(at), static_cast<int>(at >> 32) & 0xffff, static_cast<int>(size < 0xffffff00ll ? static_cast<unsigned>(size) : 0xffffff00u),
                                 0x00020000};
        int r = t / s.px, c = t % s.px;
        for (int q = wave * 64; q < tile_rows * s.px; q += 512) {
            load_to_lds(desc, c < chunks_k && r < tile_rows ? static_cast<unsigned>(r * step) + c * 16 : kNowhere, to + q * 16);
            r += down;
            c += across;
            if (c >= s.px) {
                c -= s.px;
                ++r;
            }
        }
    };
    const unsigned xs_at = lds_base, ws_at = lds_base + static_cast<unsigned>(ws - lds);
    fetch(a.weight, a.K, a.N, (chunks_n + 1) / 2 * STEP, ws_at);
    // dz's columns beyond N are zero
    for (int i = t; i < (2 * (s.a_bytes + s.b_bytes)) / 16; i += 512) reinterpret_cast<Chunk*>(das)[i] = Chunk{0, 0, 0, 0};
    __syncthreads();

    // dz: this thread's rows row, row + per_pass of a tile and its chunk of columns
    constexpr int PASSES = 2;
    const int per_pass = 512 / chunks_n, row = t / chunks_n, col = t % chunks_n * V;
    Chunk g[PASSES], e[PASSES];                                // dy; y or the kept slope, elements of the same size
    static_assert(sizeof(S) == sizeof(T), "one chunk of either");
    const auto request = [&](int64_t m0) {
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            const int r = row + p * per_pass;
            g[p] = e[p] = Chunk{0, 0, 0, 0};
            if (row >= per_pass || r >= TM || m0 + r >= a.rows) continue;
            const int64_t at = (m0 + r) * a.N + col;
            g[p] = *reinterpret_cast<const Chunk*>(a.dy + at);
            if (a.activation != kActNone) e[p] = *reinterpret_cast<const Chunk*>(static_cast<const T*>(a.kept) + at);
        }
    };
    float sums[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sums[j] = 0.0f;
    const auto place_dz = [&](int64_t m0, int buffer) {
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            const int r = row + p * per_pass;
            if (row >= per_pass || r >= TM) continue;
            typedef S SlopeVec __attribute__((ext_vector_type(V)));
            const auto dy = __builtin_bit_cast(typename Vec<T>::Type, g[p]), y = __builtin_bit_cast(typename Vec<T>::Type, e[p]);
            const auto d = __builtin_bit_cast(SlopeVec, e[p]);
            typename Vec<T>::Type z;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float f = static_cast<float>(dy[j]);
                if (a.activation == kActRelu) f *= slope<kActRelu>(static_cast<float>(y[j]));
                else if (a.activation != kActNone) f *= kept_slope(static_cast<S>(d[j]));
                if (m0 + r < a.rows) sums[j] += f;
                else f = 0.0f;
                z[j] = static_cast<T>(f);                      // (the products' operands: rounded once; the column sums are not)
            }
            const Chunk c = __builtin_bit_cast(Chunk, z);
            *reinterpret_cast<Chunk*>(das + buffer * s.a_bytes + (r * s.pa) * 16 + col / V * 16) = c;
            if constexpr (sizeof(T) == 2) *reinterpret_cast<Chunk*>(dbs + buffer * s.b_bytes + (r * s.pb) * 16 + col / V * 16) = c;
            if (a.dresidual != nullptr && m0 + r < a.rows) *reinterpret_cast<typename Vec<T>::Type*>(a.dresidual + (m0 + r) * a.N + col) = z;
        }
    };
    const auto fetch_x = [&](int64_t m0, int buffer) { fetch(a.x + m0 * a.ld_x, a.ld_x, a.rows - m0, TM, xs_at + buffer * s.x_bytes); };

    Acc16 acc[BLOCKS] = {};
    const int n_steps = (a.N + STEP - 1) / STEP;
    int buffer = 0;
    int tile = blockIdx.x;
    if (tile < a.tiles) {
        fetch_x(static_cast<int64_t>(tile) * TM, 0);
        request(static_cast<int64_t>(tile) * TM);
    }
    for (; tile < a.tiles; tile += gridDim.x, buffer ^= 1) {
        const int64_t m0 = static_cast<int64_t>(tile) * TM;
        place_dz(m0, buffer);
        settle<0>();                                           // x and dz of this tile are in LDS, and nobody reads the other buffers any more
        if (tile + static_cast<int>(gridDim.x) < a.tiles) {
            fetch_x(m0 + static_cast<int64_t>(gridDim.x) * TM, buffer ^ 1);
            request(m0 + static_cast<int64_t>(gridDim.x) * TM);
        }
        const char *x = xs + buffer * s.x_bytes, *da = das + buffer * s.a_bytes;
        const char* db = sizeof(T) == 2 ? dbs + buffer * s.b_bytes : da;
        const int pb = sizeof(T) == 2 ? s.pb : s.pa;
        if (a.dx != nullptr)
            for (int i = wave; i < TM / 32 * blocks_k; i += 8) {
                const int mb = i % (TM / 32), kb = i / (TM / 32);
                Acc16 sum = {};
#pragma unroll 4
                for (int ks = 0; ks < n_steps; ++ks) {
                    const Chunk z = *reinterpret_cast<const Chunk*>(da + ((32 * mb + l % 32) * s.pa + 2 * ks + l / 32) * 16);
                    sum = multiply_add<T>(transposed<T, true>(ws, s.px, 32 * kb, ks), z, sum);
                }
                const int64_t m = m0 + 32 * mb + l % 32;
                const int k = 32 * kb + 16 * (l / 32);
                if (m < a.rows && k < a.K) {
                    T out[16];
#pragma unroll
                    for (int r = 0; r < 16; ++r) out[r] = static_cast<T>(sum[r]);
                    store_run<T, 16>(a.dx + m * a.K + k, out, a.K - k);
                }
            }
        if (a.dweight != nullptr) {
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) {
                const int i = wave + 8 * b, nb = i / blocks_k, kb = i % blocks_k;
                if (nb >= blocks_n) continue;
#pragma unroll
                for (int ks = 0; ks < TM / STEP; ++ks)
                    acc[b] = multiply_add<T>(transposed<T, true>(x, s.px, 32 * kb, ks), transposed<T, false>(db, pb, 32 * nb, ks), acc[b]);
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (a.dweight != nullptr) {
        float* out = a.dweight + static_cast<int64_t>(blockIdx.x) * a.N * a.K;
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) {
            const int i = wave + 8 * b, n = i / blocks_k * 32 + l % 32, k = i % blocks_k * 32 + 16 * (l / 32);
            if (n >= a.N || k >= a.K) continue;
            float z[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) z[r] = acc[b][r];
            store_run<float, 16>(out + static_cast<int64_t>(n) * a.K + k, z, a.K - k);
        }
    }
    if (a.dbias != nullptr) {
        __syncthreads();                                       // (the tiles are done with: their LDS takes the sums)
        float* part = reinterpret_cast<float*>(lds);
        const int rows = narrow_sum_rows<T>(a.N, TM);          // (threads of the rows from there on hold zeros, and there is no room for them)
        if (row < rows)
#pragma unroll
            for (int j = 0; j < V; ++j) part[row * a.N + col + j] = sums[j];
        __syncthreads();
        for (int n = t; n < a.N; n += 512) {
            float f = 0.0f;
            for (int r = 0; r < rows; ++r) f += part[r * a.N + n];
            a.dbias[static_cast<int64_t>(blockIdx.x) * a.N + n] = f;
        }
    }
}

}  // namespace

}  // namespace boxconv
