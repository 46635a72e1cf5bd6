// The pointwise product y = act(x W^T + bias + residual) and its gradients for one element type (BOXCONV_INST_T: float,
// _Float16 or __bf16; compiled once for each).
#include "linear_narrow.hpp"

namespace boxconv {

namespace {

// ---- any shape, alignment and size ---------------------------------------------------------------------------
// A workgroup of four waves (2 x 2) computes a TX x TX tile; operands go through registers into LDS with every bound checked,
// the next tile's loads (of tiles of 64: the next two tiles') in flight while this one is multiplied. blockIdx.y: the part of k
// this workgroup sums. (Four groups of waves that take the tiles of k in turn, for products of few tiles, were no better: 1501 x 517
// -> 333 float16 12.4 against 13.1 us, 517 x 1501 -> 333 17.5 against 14.1 with k split over workgroups.) Bound by issue: request, shift, mask
// and store of every chunk, then the products. 1501 rows, 333 -> 517 float16 with gelu and a residual 13 us, dx 14, dW 10; 90022 rows, 431 ->
// 149 bfloat16 63 us.
template <class T, bool A_K, bool B_K, int TX>
__global__ void __launch_bounds__(256)
product_kernel(Operand<T> a, Operand<T> b, Tail<T> tail, int64_t k_part, int64_t tiles_m, int64_t tiles_n) {
    typedef TileShape<T, A_K, TX, 8> SA;
    typedef TileShape<T, B_K, TX, 8> SB;
    constexpr int F = TX / 64;                              // 32 x 32 blocks of a wave along each axis
    __shared__ Chunk lds[SA::kChunks + SB::kChunks];
    Chunk *ta = lds, *tb = lds + SA::kChunks;
    const int64_t m0 = blockIdx.x / tiles_n * TX, n0 = blockIdx.x % tiles_n * TX;
    const int64_t k_begin = blockIdx.y * k_part, k_end = min(a.depth, k_begin + k_part);
    const int wave = threadIdx.x / 64, wm = wave / 2 * (TX / 2), wn = wave % 2 * (TX / 2);
    Acc16 acc[F][F] = {};                                   // [n block][m block]
    constexpr int AHEAD = TX == 64 ? 2 : 1;
    Stage<T, A_K, TX, 256, false> sa[AHEAD];
    Stage<T, B_K, TX, 256, true> sb[AHEAD];
    const auto k_left = [&](int64_t k0) { return static_cast<int>(max<int64_t>(min<int64_t>(k_end - k0, 1 << 20), 0)); };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
        const int64_t k0 = k_begin + i * SA::KT;
        sa[i].start(a, m0, k0, AHEAD);
        sb[i].start(b, n0, k0, AHEAD);
        sa[i].request(k_left(k0));
        sb[i].request(k_left(k0));
    }
    const auto turn = [&](int64_t k0, Stage<T, A_K, TX, 256, false>& xa, Stage<T, B_K, TX, 256, true>& xb) {
        const int here = k_left(k0), later = k_left(k0 + AHEAD * SA::KT);
        xa.settle(here);
        xb.settle(here);
        __syncthreads();
        xa.store(ta);
        xb.store(tb);
        __syncthreads();
        xa.advance();
        xb.advance();
        xa.request(later);                                     // (beyond the end: one safe vector)
        xb.request(later);
#pragma unroll
        for (int ks = 0; ks < SA::kSteps; ++ks) {
            Chunk fa[F], fb[F];
#pragma unroll
            for (int j = 0; j < F; ++j) {
                fa[j] = fragment<T, A_K, TX, 8, false>(ta, wm + 32 * j, ks);
                fb[j] = fragment<T, B_K, TX, 8, true>(tb, wn + 32 * j, ks);
            }
#pragma unroll
            for (int i = 0; i < F; ++i)
#pragma unroll
                for (int j = 0; j < F; ++j) acc[i][j] = multiply_add<T>(fb[i], fa[j], acc[i][j]);
        }
    };
    for (int64_t k0 = k_begin; k0 < k_end; k0 += AHEAD * SA::KT) {
        turn(k0, sa[0], sb[0]);
        if constexpr (AHEAD == 2) {
            if (k0 + SA::KT < k_end) turn(k0 + SA::KT, sa[AHEAD - 1], sb[AHEAD - 1]);
        }
    }
    __syncthreads();
    static_assert(4 * 256 * F <= SA::kChunks + SB::kChunks, "each wave turns its sums in a part of the tiles");
    store_blocks<T, F, F>(tail, acc, m0 + wm, n0 + wn, blockIdx.y, lds + wave * 256 * F);
}

// ---- few rows ----------------------------------------------------------------------------------------------------
// y for at most 16 * MT rows: the weight is all there is to read, once. A workgroup takes 16 columns n and its waves share k, each
// with as many 16-byte loads of the weight in flight as it has; their sums meet in LDS. (16 x 16 matrix instructions: the weight's
// rows are the first operand, so that a lane ends up with four consecutive n of one row.)
typedef float Acc4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ Acc4 multiply_add16(Chunk b, Chunk a, Acc4 c, __bf16) {
    typedef __bf16 Eight __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(Eight, b), __builtin_bit_cast(Eight, a), c, 0, 0, 0);
}
__device__ __forceinline__ Acc4 multiply_add16(Chunk b, Chunk a, Acc4 c, _Float16) {
    typedef _Float16 Eight __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(Eight, b), __builtin_bit_cast(Eight, a), c, 0, 0, 0);
}
__device__ __forceinline__ Acc4 multiply_add16(Chunk b, Chunk a, Acc4 c, float) {
    const Acc4 x = __builtin_bit_cast(Acc4, b), y = __builtin_bit_cast(Acc4, a);
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
    return c;
}

template <class T, int MT>
__global__ void __launch_bounds__(1024)
few_rows_kernel(Operand<T> a, Operand<T> b, Tail<T> tail) {
    constexpr int V = Vec<T>::kLen, STEP = 4 * V, U = MT == 1 ? 8 : 4;     // k of one load of a wave; loads in flight
    extern __shared__ Acc4 sums[];
    const int l = threadIdx.x % 64, wave = threadIdx.x / 64, waves = blockDim.x / 64;
    const int64_t n0 = blockIdx.x * 16ll, n = n0 + l % 16;
    const int64_t steps = (a.depth + STEP - 1) / STEP, part = (steps + waves - 1) / waves;
    const int64_t first = wave * part, last = min(steps, first + part);
    Acc4 acc[MT] = {};
    // (rows beyond the end repeat the last one: nobody stores their sums)
    const T *w_row = b.p + min(n, b.extent - 1) * b.ld + l / 16 * V, *x_row[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) x_row[i] = a.p + min<int64_t>(16 * i + l % 16, a.extent - 1) * a.ld + l / 16 * V;
    int64_t s = first;
    for (; s + U <= last && (s + U) * STEP <= a.depth; s += U) {
        Chunk w[U], x[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            w[u] = __builtin_bit_cast(Chunk, *reinterpret_cast<const typename Vec<T>::Type*>(w_row + s * STEP + u * STEP));
#pragma unroll
            for (int i = 0; i < MT; ++i) x[u][i] = __builtin_bit_cast(Chunk, *reinterpret_cast<const typename Vec<T>::Type*>(x_row[i] + s * STEP + u * STEP));
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[i] = multiply_add16(w[u], x[u][i], acc[i], T());
    }
#pragma unroll 1
    for (; s < last; ++s) {
        const int64_t valid = a.depth - (s * STEP + l / 16 * V);
        Chunk w = request_chunk(w_row + s * STEP, valid, b.p), x[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) x[i] = request_chunk(x_row[i] + s * STEP, valid, a.p);
        settle_chunk<T>(w, valid);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            settle_chunk<T>(x[i], valid);
            acc[i] = multiply_add16(w, x[i], acc[i], T());
        }
    }
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

// The same for operands of whole aligned chunks: fragments read straight from memory touch another cache line with every lane,
// and the address units take one line a cycle (16 rows of 4096 float16 through 1024 columns: 10.6 us). Here every wave brings
// 512 bytes of k of its rows to LDS as they lie in memory, then reads its fragments there; chunk c of row r at c ^ r keeps
// the 16 rows of an access in different banks. 6.2 us that way; one row through 1024 -> 4096 bfloat16 (8.4 MB of weight) 4.3 us, 1.9 TB/s:
// a launch, one round trip to memory and the join of the waves.
template <class T, int MT>
__global__ void __launch_bounds__(512)
few_whole_rows_kernel(Operand<T> a, Operand<T> b, Tail<T> tail) {
    constexpr int V = Vec<T>::kLen, BLOCK = 32 * V, kRows = 16 * (MT + 1); // values of k in a block; rows of the weight, then of x
    extern __shared__ Chunk blocks[];
    const int l = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), waves = blockDim.x / 64;
    const int64_t n0 = blockIdx.x * 16ll;
    const int depth = static_cast<int>(a.depth), count = (depth + BLOCK - 1) / BLOCK, part = (count + waves - 1) / waves;
    const Chunk* mine = blocks + wave * kRows * 32;
    const unsigned to = static_cast<unsigned>(reinterpret_cast<uintptr_t>((LdsVoid)mine));
    const auto describe = [](const T* p, int64_t elements) {
        const uint64_t at = reinterpret_cast<uint64_t>(p);
        const int64_t size = elements * static_cast<int64_t>(sizeof(T));
        return Descriptor{static_cast<int>(at), static_cast<int>(at >> 32) & 0xffff, static_cast<int>(size < 0xffffff00ll ? static_cast<unsigned>(size) : 0xffffff00u), 0x00020000};
    };
    const int rows_w = static_cast<int>(min<int64_t>(16, b.extent - n0)), rows_x = static_cast<int>(a.extent);
    const Descriptor dw = describe(b.p + n0 * b.ld, (rows_w - 1) * b.ld + depth), dx = describe(a.p, (rows_x - 1) * a.ld + depth);
    Acc4 acc[MT] = {};
    for (int s = wave * part; s < min(count, (wave + 1) * part); ++s) {
#pragma unroll
        for (int i = 0; i < kRows / 2; ++i) {                  // two rows at a time
            const int r = 2 * i + l / 32, c = l % 32 ^ (r & 15), k = s * BLOCK + c * V, row = i < 8 ? r : r - 16;
            const bool inside = k < depth && row < (i < 8 ? rows_w : rows_x);
            const int64_t ld = i < 8 ? b.ld : a.ld;
            load_to_lds(i < 8 ? dw : dx, inside ? static_cast<unsigned>((row * ld + k) * static_cast<int64_t>(sizeof(T))) : kNowhere, to + i * 1024);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // (a wave's blocks are its own)
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
            const int r = l % 16, c = 4 * ks + l / 16 ^ r;
            const Chunk w = mine[r * 32 + c];
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[i] = multiply_add16(w, mine[(16 + 16 * i + r) * 32 + c], acc[i], T());
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");     // read before the next block overwrites them
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

// Column sums of `bands` rows of `cols` floats, WIDE columns at a time (all, or `most` from `sums` on), the other threads side by
// side down the rows: an order that only the shapes decide. part: a float per thread.
template <class T, int WIDE>
__device__ __forceinline__ void join_columns(float* part, const float* sums, T* out, int64_t cols, int bands, int64_t most = -1) {
    const int x = threadIdx.x % WIDE, row = threadIdx.x / WIDE, rows = blockDim.x / WIDE;
    if (most < 0) most = cols;
    for (int64_t c0 = 0; c0 < most; c0 += WIDE) {
        const int64_t c = c0 + x;
        float s = 0.0f;
        if (c < most) {
#pragma unroll 8
            for (int i = row; i < bands; i += rows) s += sums[i * cols + c];
        }
        part[threadIdx.x] = s;
        __syncthreads();
        for (int half = rows / 2; half > 0; half >>= 1) {
            if (row < half) part[threadIdx.x] = s += part[threadIdx.x + half * WIDE];
            __syncthreads();
        }
        if (row == 0 && c < most) out[c] = static_cast<T>(s);
    }
}

// The parts of a split product, added in an order that only the shape decides, and the tail. A workgroup takes 256 / `lanes`
// runs of eight columns; `lanes` (a power of two) threads share the parts of a run. Bound by reading the parts where there are many: 16 x
// 1024 x 1024 floats 8 us; 3 to 6 us, the launch, in small products.
template <class T>
__global__ void __launch_bounds__(256) join_parts_kernel(Tail<T> tail, int splits, int64_t runs_per_row, int64_t runs, int lanes, const float* sums, T* dbias) {
    __shared__ float part[256][9];
    if (sums != nullptr && blockIdx.x == gridDim.x - 1) {              // the last workgroup: column sums of the same parts
        join_columns<T, 32>(&part[0][0], sums, dbias, tail.rows, splits);
        return;
    }
    const int per = 256 / lanes, lane = threadIdx.x / per;
    const int64_t id = blockIdx.x * static_cast<int64_t>(per) + threadIdx.x % per;
    const int64_t m = id / runs_per_row, n = id % runs_per_row * 8;
    float z[8] = {};
    if (id < runs) {
        const float* p = tail.partial + m * tail.cols + n;
#pragma unroll 4
        for (int s = lane; s < splits; s += lanes) {
            float v[8];
            load_run<float, 8>(p + s * tail.rows * tail.cols, v, tail.cols - n);
#pragma unroll
            for (int i = 0; i < 8; ++i) z[i] += v[i];
        }
    }
    if (lanes > 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) part[threadIdx.x][i] = z[i];
        for (int half = lanes / 2; half > 0; half >>= 1) {
            __syncthreads();
            if (lane < half) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    z[i] += part[threadIdx.x + half * per][i];
                    part[threadIdx.x][i] = z[i];
                }
            }
        }
    }
    if (lane == 0 && id < runs) apply_tail<T, 8>(tail, z, m, n);
}

// ---- dz = dy * act'(z), and its column sums ---------------------------------------------------------------------
// A workgroup takes 256 columns (8 per thread, 32 threads) of a band of rows, 8 rows at a time. sums: [bands][cols], null
// if not wanted; dz: null if not wanted. kept: y for relu, the kept slope for silu and gelu. Bound by memory: 8192 x 2048 bfloat16 (101 MB)
// 22 us, 4.5 TB/s. dz is rounded to T here, once, for both products: with 16-bit types these are the matrix instructions' operands, and dz in two
// parts would double the backward's matrix work. dx and dW of silu and gelu are then 1.4 times as far from 64 bits as with dz in float: 0.0024 of
// their norm instead of 0.0017 in bfloat16 (8192 x 4096 -> 2048), 0.00029 instead of 0.00021 in float16 (1501 x 333 -> 517). The column sums take it unrounded.
template <class T>
__global__ void __launch_bounds__(256)
slope_kernel(const T* __restrict__ dy, const void* __restrict__ kept, T* __restrict__ dz, float* __restrict__ sums, T* __restrict__ dbias, int64_t rows,
             int64_t cols, int64_t band, int activation) {
    typedef typename SlopeOf<T>::Type S;
    __shared__ float part[8][256];
    const int64_t n = blockIdx.y * 256ll + threadIdx.x % 32 * 8, first = blockIdx.x * band, last = min(rows, first + band);
    const int64_t valid = cols - n;
    float sum[8] = {};
    for (int64_t m = first + threadIdx.x / 32; m < last; m += 8) {
        if (valid <= 0) break;
        T g[8];
        load_run<T, 8>(dy + m * cols + n, g, valid);
        float d[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = static_cast<float>(g[i]);
        if (activation == kActRelu) {
            T y[8];
            load_run<T, 8>(static_cast<const T*>(kept) + m * cols + n, y, valid);
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] *= slope<kActRelu>(static_cast<float>(y[i]));
        } else if (activation != kActNone) {
            S s[8];
            load_run<S, 8>(static_cast<const S*>(kept) + m * cols + n, s, valid);
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] *= kept_slope(s[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            sum[i] += d[i];
            g[i] = static_cast<T>(d[i]);
        }
        if (dz != nullptr) store_run<T, 8>(dz + m * cols + n, g, valid);
    }
    if (sums == nullptr) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) part[threadIdx.x / 32][threadIdx.x % 32 * 8 + i] = sum[i];
    __syncthreads();
    const int64_t col = blockIdx.y * 256ll + threadIdx.x;
    if (col < cols) {
        float s = 0.0f;
        for (int r = 0; r < 8; ++r) s += part[r][threadIdx.x];
        if (gridDim.x == 1) dbias[col] = static_cast<T>(s);            // (one band: nothing to join)
        else sums[blockIdx.x * cols + col] = s;
    }
}

template <class T>
__global__ void __launch_bounds__(1024) join_bias_kernel(const float* __restrict__ sums, T* __restrict__ dbias, int64_t cols, int bands) {
    __shared__ float part[1024];
    join_columns<T, 16>(part, sums + blockIdx.x * 16ll, dbias + blockIdx.x * 16ll, cols, bands, std::min<int64_t>(16, cols - blockIdx.x * 16ll));
}

// ---- plans ---------------------------------------------------------------------------------------------------------
size_t round_up(size_t v) { return (v + 255) / 256 * 256; }

struct ProductPlan {
    int shape, splits;         // shape: which of the kernels below
    int64_t k_part, tiles_m, tiles_n;
    size_t partial_bytes;
};

// The kernels' tiles, and what they take a compute unit that holds `w` of their workgroups, in us: a step of 128 bytes of k fixed + each * w
// (float: each_float), a workgroup's start and epilogue as long as `ends` steps, and `slope` for an epilogue that keeps act' on a full unit.
// Measured on bfloat16 products, M x N x K: 8192 x 4096 x 2048 takes 107 us with 256 x 256 tiles, 137 with 128 x 128; 2048 x 2048 x
// 4096 takes 78, 48 and, with 64 x 64, 52; 512 x 512 x 4096 33 with 128 x 128, 36 with 64 x 64 (none of them split). Short k, the same
// three: 300000 x 256 x 64 68, 76 and 86 us; 380192 x 160 x 32 with a kept slope 137, 149 and 109; float, 48552 x 456 x 208 with one 185, 158
// and 145. Tiles of 256 x 128 were no better than 128 x 128 anywhere: their waves read as much from LDS per product. All of these have k contiguous
// in both operands. For the weight gradient, where it is the slow index of both, the costs promise too little: 8192 x 4096 -> 2048 with 128 x 128 tiles 119
// us, and it takes 136 alone and 164 in a training step; other tiles and splits have not been measured there.
struct ProductShape { int tm, tn, resident; double fixed, each, each_float, ends, slope; };
constexpr ProductShape kWide[] = {{256, 256, 1, 0.0, 1.38, 7.2, 8.7, 10.0}, {128, 128, 2, 0.46, 0.21, 1.8, 7.6, 5.0}, {64, 64, 4, 0.44, 0.075, 0.44, 5.0, 1.6}};
constexpr ProductShape kAny[] = {{128, 128, 2, 0.8, 0.4, 2.0, 7.0, 5.0}, {64, 64, 4, 0.5, 0.15, 0.5, 7.0, 1.6}};

// The tile and the number of parts of k that promise the shortest time: rounds of workgroups, and the parts' way through memory at 4 TB/s
// with one more launch.
template <class T, int N>
ProductPlan plan_product(const ProductShape (&shapes)[N], int64_t m, int64_t n, int64_t k, bool keeps_slope) {
    constexpr int KT = 8 * Vec<T>::kLen;
    ProductPlan best = {};
    double least = 0.0;
    const int64_t steps = std::max<int64_t>((k + KT - 1) / KT, 1);
    for (int i = 0; i < N; ++i) {
        const ProductShape& s = shapes[i];
        const int64_t tm = (m + s.tm - 1) / s.tm, tn = (n + s.tn - 1) / s.tn, tiles = std::max<int64_t>(tm * tn, 1);
        for (int64_t splits = 1; splits <= 256 && splits * 2 <= std::max<int64_t>(steps, 2); splits *= 2) {
            const int64_t part = (steps + splits - 1) / splits, parts = (steps + part - 1) / part, groups = tiles * parts;
            const int64_t slots = 256 * s.resident, rounds = (groups + slots - 1) / slots;
            const double w = groups >= slots ? s.resident : static_cast<double>((groups + 255) / 256);
            double t = static_cast<double>(part) * (s.fixed + (sizeof(T) == 4 ? s.each_float : s.each) * w) + s.ends * (s.fixed + s.each * w);
            if (keeps_slope && parts == 1) t += s.slope * w / s.resident;
            t *= static_cast<double>(rounds);
            if (parts > 1) t += 4.0 + static_cast<double>(parts) * static_cast<double>(m) * static_cast<double>(n) * 8.0 / 4e6;
            if (best.splits == 0 || t < least) {
                least = t;
                best = {i, static_cast<int>(parts), part * KT, tm, tn, parts > 1 ? static_cast<size_t>(parts) * m * n * 4 : 0};
            }
            if (groups >= 1024) break;
        }
    }
    return best;
}

// Whether tiles of this operand can come straight into LDS: whole aligned chunks, offsets within a tile in 31 bits. With k as the slow index
// rows must not overlap either (an expanded input's lie on top of each other): rows beyond the last one are zeros only because they lie beyond the
// operand's end, and others' values there would be multiplied by the other operand's zeros, which gives NaN where they are infinite.
template <class T, bool K_MAJOR>
bool whole_chunks(const Operand<T>& o) {
    constexpr int V = Vec<T>::kLen;
    return reinterpret_cast<uintptr_t>(o.p) % 16 == 0 && o.ld % V == 0 && (K_MAJOR ? o.depth : o.extent) % V == 0 && o.depth < (int64_t(1) << 30) &&
           o.ld < (int64_t(1) << 31) / (256 * static_cast<int64_t>(sizeof(T))) && (K_MAJOR || o.ld >= o.extent);
}

template <class T, bool A_K, bool B_K, int TM, int TN, int WM, int WN>
void launch_wide(const char* name, const Operand<T>& a, const Operand<T>& b, const Tail<T>& tail, const ProductPlan& p, hipStream_t stream) {
    constexpr size_t lds = kRing * sizeof(Chunk) * (TileShape<T, A_K, TM, 8>::kChunks + TileShape<T, B_K, TN, 8>::kChunks);
    const dim3 grid(static_cast<unsigned>(p.tiles_m * p.tiles_n), p.splits);
    BOXCONV_LAUNCH(name, (product_wide_kernel<T, A_K, B_K, TM, TN, WM, WN>), grid, dim3(WM * WN * 64), lds, stream, a, b, tail, p.k_part,
                   static_cast<unsigned>(p.tiles_m), static_cast<unsigned>(p.tiles_n));
}

template <class T>
void join_parts(const Tail<T>& tail, int splits, hipStream_t stream, const float* sums = nullptr, T* dbias = nullptr) {
    const int64_t per_row = (tail.cols + 7) / 8, runs = per_row * tail.rows;
    int lanes = 1;                                         // threads for every CU, and at least four parts for each
    while (lanes < 64 && lanes * 8 <= splits && runs * lanes < 65536) lanes *= 2;
    const int64_t per = 256 / lanes;
    BOXCONV_LAUNCH("join_parts", (join_parts_kernel<T>), dim3(static_cast<unsigned>((runs + per - 1) / per + (sums != nullptr))), dim3(256), 0, stream, tail, splits,
                   per_row, runs, lanes, sums, dbias);
}

template <class T, int MT>
hipError_t few_rows(const Operand<T>& a, const Operand<T>& b, const Tail<T>& tail, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>((tail.cols + 15) / 16));
    int waves = 1;
    if (whole_chunks<T, true>(a) && whole_chunks<T, true>(b) && a.ld >= a.depth && a.depth < (1 << 28)) {
        constexpr int BLOCK = 32 * Vec<T>::kLen;
        while (waves < (MT == 1 ? 8 : 4) && waves * BLOCK < a.depth) waves *= 2;
        BOXCONV_LAUNCH("linear_few_rows", (few_whole_rows_kernel<T, MT>), grid, dim3(waves * 64), static_cast<size_t>(waves) * 16 * (MT + 1) * 512, stream, a, b, tail);
        return hipGetLastError();
    }
    constexpr int STEP = 4 * Vec<T>::kLen;
    for (waves = 4; waves < 16 && waves * 8 * STEP < a.depth;) waves *= 2;    // waves with 8 loads each
    BOXCONV_LAUNCH("linear_few_rows", (few_rows_kernel<T, MT>), grid, dim3(waves * 64), static_cast<size_t>(waves) * MT * 1024, stream, a, b, tail);
    return hipGetLastError();
}

template <class T, bool A_K, bool B_K>
void launch_product(const char* name, Operand<T> a, const Operand<T>& b, Tail<T> tail, ProductPlan p, bool wide, hipStream_t stream) {
    // a grid has fewer than 2^32 threads: with more tiles (never in several parts of k) some rows of the output after the others
    const int64_t threads = wide && p.shape == 0 ? 512 : 256, tile = wide ? kWide[p.shape].tm : kAny[p.shape].tm;
    const int64_t rows = tail.rows, most = std::max<int64_t>(1, kMostThreads / threads / p.tiles_n) * tile;
    for (int64_t m = 0; m < rows; m += most) {
        tail.rows = a.extent = std::min(most, rows - m);
        p.tiles_m = (tail.rows + tile - 1) / tile;
        if (wide) {
            switch (p.shape) {
                case 0: launch_wide<T, A_K, B_K, 256, 256, 4, 2>(name, a, b, tail, p, stream); break;
                case 1: launch_wide<T, A_K, B_K, 128, 128, 2, 2>(name, a, b, tail, p, stream); break;
                default: launch_wide<T, A_K, B_K, 64, 64, 2, 2>(name, a, b, tail, p, stream);
            }
        } else {
            const dim3 grid(static_cast<unsigned>(p.tiles_m * p.tiles_n), p.splits);
            if (p.shape == 0) BOXCONV_LAUNCH(name, (product_kernel<T, A_K, B_K, 128>), grid, dim3(256), 0, stream, a, b, tail, p.k_part, p.tiles_m, p.tiles_n);
            else BOXCONV_LAUNCH(name, (product_kernel<T, A_K, B_K, 64>), grid, dim3(256), 0, stream, a, b, tail, p.k_part, p.tiles_m, p.tiles_n);
        }
        a.p += most * (A_K ? a.ld : 1);
        tail.out += most * tail.cols;
        if (tail.residual != nullptr) tail.residual += most * tail.ld_residual;
        if (tail.slope != nullptr) tail.slope += most * tail.cols;
    }
}

template <class T, bool A_K, bool B_K>
hipError_t product(const char* name, Operand<T> a, Operand<T> b, Tail<T> tail, float* workspace, hipStream_t stream) {
    const bool wide = whole_chunks<T, A_K>(a) && whole_chunks<T, B_K>(b);
    const bool keeps = tail.slope != nullptr;
    const ProductPlan p = wide ? plan_product<T>(kWide, tail.rows, tail.cols, a.depth, keeps) : plan_product<T>(kAny, tail.rows, tail.cols, a.depth, keeps);
    tail.partial = p.splits > 1 ? workspace : nullptr;
    launch_product<T, A_K, B_K>(name, a, b, tail, p, wide, stream);
    if (p.splits > 1) join_parts(tail, p.splits, stream);
    return hipGetLastError();
}

template <class T>
size_t product_workspace(int64_t m, int64_t n, int64_t k) {
    size_t most = 0;
    for (const bool keeps : {false, true})
        most = std::max({most, plan_product<T>(kWide, m, n, k, keeps).partial_bytes, plan_product<T>(kAny, m, n, k, keeps).partial_bytes});
    return most;
}


struct BandPlan { int64_t band; int bands; };
BandPlan plan_bands(int64_t rows, int64_t cols) {
    const int64_t across = (cols + 255) / 256;
    int64_t bands = std::max<int64_t>(1, std::min<int64_t>((1024 + across - 1) / across, rows <= 256 ? 1 : (rows + 31) / 32));
    BandPlan p;
    p.band = (rows + bands - 1) / bands;
    p.band = std::max<int64_t>(8, (p.band + 7) / 8 * 8);
    p.bands = static_cast<int>((rows + p.band - 1) / p.band);
    return p;
}

// ---- few channels --------------------------------------------------------------------------------------------------
struct NarrowPlan {
    bool applies;
    int tm, blocks, workgroups, tiles;
    size_t lds, bytes;         // of LDS; of the partial sums
};

// Sizes that narrow_grad_kernel covers. Two tiles at least for a workgroup, while there are few.
template <class T>
NarrowPlan plan_narrow(int64_t rows, int64_t K, int64_t N) {
    constexpr int V = Vec<T>::kLen;
    NarrowPlan p = {};
    if (K < V || N < V || K % V || N % V || K > 1024 || N > 128 || rows > (int64_t(1) << 36)) return p;
    const int blocks = static_cast<int>((K + 31) / 32 * ((N + 31) / 32));
    p.blocks = 1;
    while (p.blocks * 8 < blocks) p.blocks *= 2;
    if (p.blocks > 4) return p;
    for (p.tm = sizeof(T) == 2 ? 64 : 32; p.tm >= 32; p.tm /= 2) {
        p.lds = static_cast<size_t>(narrow_lds<T>(static_cast<int>(N), static_cast<int>(K), p.tm).total());
        if (p.lds <= kMaxDynamicLds && 2 * (512 / static_cast<int>(N / V)) >= p.tm) break;
    }
    if (p.tm < 32) return p;
    const int64_t tiles = (rows + p.tm - 1) / p.tm;
    const int64_t resident = std::min<int64_t>(2, static_cast<int64_t>(kMaxDynamicLds / p.lds)) * 256;
    if (tiles > (int64_t(1) << 30) || tiles < 1) return p;
    p.tiles = static_cast<int>(tiles);
    p.workgroups = static_cast<int>(std::min(resident, (tiles + 1) / 2));
    p.bytes = round_up(static_cast<size_t>(p.workgroups) * N * K * 4) + static_cast<size_t>(p.workgroups) * N * 4;
    p.applies = true;
    return p;
}

template <class T, int TM>
void launch_narrow(const NarrowArgs<T>& a, const NarrowPlan& p, hipStream_t stream) {
    const dim3 grid(p.workgroups), block(512);
    if (p.blocks == 1) BOXCONV_LAUNCH("linear_narrow_grad", (narrow_grad_kernel<T, TM, 1>), grid, block, p.lds, stream, a);
    else if (p.blocks == 2) BOXCONV_LAUNCH("linear_narrow_grad", (narrow_grad_kernel<T, TM, 2>), grid, block, p.lds, stream, a);
    else BOXCONV_LAUNCH("linear_narrow_grad", (narrow_grad_kernel<T, TM, 4>), grid, block, p.lds, stream, a);
}

template <class T>
hipError_t narrow_backward(const LinearGradCall& c, const NarrowPlan& p, void* workspace, hipStream_t stream) {
    NarrowArgs<T> a = {};
    a.x = static_cast<const T*>(c.x);
    a.weight = static_cast<const T*>(c.weight);
    a.dy = static_cast<const T*>(c.dy);
    a.kept = c.kept;
    a.ld_x = c.ld_x;
    a.rows = c.rows;
    a.dx = static_cast<T*>(c.dx);
    a.dresidual = static_cast<T*>(c.dresidual);
    a.N = static_cast<int>(c.N);
    a.K = static_cast<int>(c.K);
    a.activation = c.activation;
    a.tiles = p.tiles;
    float* parts = static_cast<float*>(workspace);
    float* sums = parts + round_up(static_cast<size_t>(p.workgroups) * c.N * c.K * 4) / 4;
    a.dweight = c.dweight ? parts : nullptr;
    a.dbias = c.dbias ? sums : nullptr;
    if (p.tm == 64) launch_narrow<T, 64>(a, p, stream);
    else launch_narrow<T, 32>(a, p, stream);
    if (c.dweight != nullptr) {
        Tail<T> tail = {};
        tail.out = static_cast<T*>(c.dweight);
        tail.rows = c.N;
        tail.cols = c.K;
        tail.partial = parts;
        join_parts(tail, p.workgroups, stream, a.dbias, static_cast<T*>(c.dbias));
    } else if (c.dbias != nullptr)
        BOXCONV_LAUNCH("join_bias", (join_bias_kernel<T>), dim3(static_cast<unsigned>((c.N + 15) / 16)), dim3(1024), 0, stream, sums, static_cast<T*>(c.dbias), c.N,
                       p.workgroups);
    return hipGetLastError();
}

}  // namespace

template <class T>
size_t linear_forward_workspace(int64_t rows, int64_t K, int64_t N) { return product_workspace<T>(rows, N, K); }

// [dz, unless the residual's gradient holds it][column sums per band][parts of a split product]
template <class T>
size_t linear_backward_workspace(int64_t rows, int64_t K, int64_t N) {
    return std::max(plan_narrow<T>(rows, K, N).bytes,
                    round_up(static_cast<size_t>(rows) * N * sizeof(T)) + round_up(static_cast<size_t>(plan_bands(rows, N).bands) * N * 4) +
                        std::max(product_workspace<T>(rows, K, N), product_workspace<T>(N, K, rows)));
}

template <class T>
hipError_t linear_forward(const LinearCall& c, void* workspace, hipStream_t stream) {
    const Operand<T> a = {static_cast<const T*>(c.x), c.ld_x, c.rows, c.K};
    const Operand<T> b = {static_cast<const T*>(c.weight), c.K, c.N, c.K};
    Tail<T> tail = {};
    tail.out = static_cast<T*>(c.y);
    tail.rows = c.rows;
    tail.cols = c.N;
    tail.bias = static_cast<const T*>(c.bias);
    tail.residual = static_cast<const T*>(c.residual);
    tail.ld_residual = c.ld_residual;
    tail.slope = static_cast<typename SlopeOf<T>::Type*>(c.slope);
    tail.activation = c.activation;
    if (c.rows <= 16 && c.K >= Vec<T>::kLen) return few_rows<T, 1>(a, b, tail, stream);
    if (c.rows <= 32 && c.K >= Vec<T>::kLen) return few_rows<T, 2>(a, b, tail, stream);
    return product<T, true, true>("linear", a, b, tail, static_cast<float*>(workspace), stream);
}

template <class T>
hipError_t linear_backward(const LinearGradCall& c, void* workspace, hipStream_t stream) {
    const NarrowPlan narrow = plan_narrow<T>(c.rows, c.K, c.N);
    const auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    if (narrow.applies && (c.dx != nullptr || c.dweight != nullptr) && c.x != nullptr && c.weight != nullptr && aligned(c.x) && aligned(c.weight) &&
        aligned(c.dy) && aligned(c.kept) && c.ld_x % Vec<T>::kLen == 0 && c.ld_x >= c.K && c.ld_x < (int64_t(1) << 24))
        return narrow_backward<T>(c, narrow, workspace, stream);
    char* ws = static_cast<char*>(workspace);
    T* scratch = reinterpret_cast<T*>(ws);
    ws += round_up(static_cast<size_t>(c.rows) * c.N * sizeof(T));
    const BandPlan bands = plan_bands(c.rows, c.N);
    float* sums = reinterpret_cast<float*>(ws);
    ws += round_up(static_cast<size_t>(bands.bands) * c.N * 4);
    float* parts = reinterpret_cast<float*>(ws);
    const T* dy = static_cast<const T*>(c.dy);
    const T* dz = dy;
    T* write = static_cast<T*>(c.dresidual);
    if (c.activation != kActNone) {
        if (write == nullptr && (c.dx != nullptr || c.dweight != nullptr)) write = scratch;
        dz = write;
    }
    if (write != nullptr || c.dbias != nullptr) {
        const dim3 grid(bands.bands, static_cast<unsigned>((c.N + 255) / 256));
        BOXCONV_LAUNCH("linear_slope", (slope_kernel<T>), grid, dim3(256), 0, stream, dy, c.kept, write, c.dbias ? sums : nullptr,
                       static_cast<T*>(c.dbias), c.rows, c.N, bands.band,
                       c.activation);
        if (c.dbias != nullptr && bands.bands > 1)
            BOXCONV_LAUNCH("join_bias", (join_bias_kernel<T>), dim3(static_cast<unsigned>((c.N + 15) / 16)), dim3(1024), 0, stream, sums, static_cast<T*>(c.dbias),
                           c.N, bands.bands);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    Tail<T> tail = {};
    if (c.dx != nullptr) {
        tail.out = static_cast<T*>(c.dx);
        tail.rows = c.rows;
        tail.cols = c.K;
        const Operand<T> a = {dz, c.N, c.rows, c.N};
        const Operand<T> b = {static_cast<const T*>(c.weight), c.K, c.K, c.N};
        if (const hipError_t e = product<T, true, false>("linear_dx", a, b, tail, parts, stream); e != hipSuccess) return e;
    }
    if (c.dweight != nullptr) {
        tail.out = static_cast<T*>(c.dweight);
        tail.rows = c.N;
        tail.cols = c.K;
        const Operand<T> a = {dz, c.N, c.N, c.rows};
        const Operand<T> b = {static_cast<const T*>(c.x), c.ld_x, c.K, c.rows};
        if (const hipError_t e = product<T, false, false>("linear_dweight", a, b, tail, parts, stream); e != hipSuccess) return e;
    }
    return hipSuccess;
}

template size_t linear_forward_workspace<BOXCONV_INST_T>(int64_t, int64_t, int64_t);
template size_t linear_backward_workspace<BOXCONV_INST_T>(int64_t, int64_t, int64_t);
template hipError_t linear_forward<BOXCONV_INST_T>(const LinearCall&, void*, hipStream_t);
template hipError_t linear_backward<BOXCONV_INST_T>(const LinearGradCall&, void*, hipStream_t);

}  // namespace boxconv
