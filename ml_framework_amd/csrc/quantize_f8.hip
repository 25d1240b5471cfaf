// quantize_f8.hip -- a weight matrix in 8 bits (seera_hip_quantize_weights_f8):
// codes [n][k padded to 128], a scale for each 128 x 128 of them.
//
// A block of threads has a tile of 128 x 128 in its registers: read once, its
// largest value found, its codes written. A thread holds 16 values along k of four
// columns of n (or, of a matrix that lies as [n, k], 16 values of k of four rows), so
// that the 16-byte stores of 8 lanes are 128 bytes of memory next to each other and
// nothing goes through shared memory. 256 threads of four columns, not 1024 of one:
// a compute unit then holds tiles that load beside tiles that store.
//
// 12288 x 4096 bf16, 151 MB moved, in 34 us (4.5 TB/s; a copy of this size reaches 5
// to 7): bound by memory. It took 58 with 1024 threads a tile, 51 with 256, 48 with
// codes stored past the caches (the tile's 128 lines are 4096 bytes apart), and 34
// once the largest of 16-bit values is found by their bits, two at a time: a
// conversion and a comparison for each value had kept the vector units as busy as the
// memory.
#include "f8.h"
#include "inference.h"
#include "io_types.h"
#include "runtime.h"

namespace seera {
namespace {

typedef uint32_t Codes __attribute__((ext_vector_type(4)));

template <class T, int COUNT>
struct Piece {
    static constexpr int N = COUNT;
    T v[N];
};
// N values from column c of a row of `cols`; zeros past its end.
template <int N, class T>
__device__ __forceinline__ Piece<T, N> piece(const T* row, int c, int cols) {
    Piece<T, N> p;
    if (c + N <= cols) {
        __builtin_memcpy(&p, row + c, sizeof(p));
        return p;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) p.v[i] = c + i < cols ? row[c + i] : from_f32<T>(0.f);
    return p;
}

// The largest magnitude of pieces, as the bits of an fp32 value: of 16-bit values two at a
// time, as their bits have the order of their magnitudes.
template <class T>
struct Largest {
    uint32_t bits = 0;
    template <int N>
    __device__ __forceinline__ void take(const Piece<T, N>& p) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < N; ++i) bits = max(bits, magnitude(p.v[i]));
        } else {
            typedef uint16_t Two __attribute__((ext_vector_type(2)));
            uint32_t w[N / 2];
            __builtin_memcpy(w, &p, sizeof(p));
#pragma unroll
            for (int i = 0; i < N / 2; ++i)
                bits = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(Two, bits), __builtin_bit_cast(Two, w[i] & 0x7fff7fffu)));
        }
    }
    __device__ __forceinline__ uint32_t value() const {
        if constexpr (sizeof(T) == 4) return bits;
        else return magnitude(to_f32(__builtin_bit_cast(T, (uint16_t)max(bits & 0xffffu, bits >> 16))));
    }
};

// The largest of the block's values, in all threads.
template <int WAVES>
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* part) {
#pragma unroll
    for (int m = 32; m; m >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, m));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) v = max(v, part[w]);
    return v;
}

// Matrices that lie as [k, n]. Lane 8 c + r has k = 16 r .. 16 r + 15 and the c-th
// four of a wave's 32 columns.
template <class T>
__global__ __launch_bounds__(256) void quantize_columns(QuantizeF8 a) {
    constexpr int N = 4, WAVES = 4;
    __shared__ uint32_t part[WAVES];
    const int blocks = (int)(f8_padded(a.k) / kF8Block);
    const int kb = blockIdx.x % blocks, nb = blockIdx.x / blocks;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int k0 = kb * kF8Block + (lane & 7) * 16, n0 = nb * kF8Block + (wave * 8 + (lane >> 3)) * N;
    Piece<T, N> v[16];
    Largest<T> largest;
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = piece<N>((const T*)a.w + min(k0 + j, a.k - 1) * a.ldw, n0, a.n);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (k0 + j >= a.k) v[j].v[i] = from_f32<T>(0.f);
        largest.take(v[j]);
    }
    const F8Scale f(block_max<WAVES>(largest.value(), part));
    if (threadIdx.x == 0) a.scales[(int64_t)nb * blocks + kb] = f.scale;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (n0 + i >= a.n) continue;
        Codes w;
#pragma unroll
        for (int q = 0; q < 4; ++q)
            w[q] = f8_codes(f.quotient(to_f32(v[4 * q].v[i])), f.quotient(to_f32(v[4 * q + 1].v[i])), f.quotient(to_f32(v[4 * q + 2].v[i])),
                             f.quotient(to_f32(v[4 * q + 3].v[i])));
        __builtin_nontemporal_store(w, (Codes*)(a.codes + (int64_t)(n0 + i) * blocks * kF8Block + k0));
    }
}

// Matrices that lie as [n, k]: lane 8 c + r has 16 values k = 16 r .. of each of
// eight rows, four waves of 8 rows four times.
template <class T>
__global__ __launch_bounds__(256) void quantize_rows(QuantizeF8 a) {
    constexpr int N = 16 / sizeof(T), PIECES = 16 / N;
    __shared__ uint32_t part[4];
    const int blocks = (int)(f8_padded(a.k) / kF8Block);
    const int kb = blockIdx.x % blocks, nb = blockIdx.x / blocks;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int k0 = kb * kF8Block + (lane & 7) * 16, n0 = nb * kF8Block + wave * 32 + (lane >> 3);
    Piece<T, N> v[4][PIECES];
    Largest<T> largest;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < PIECES; ++i) v[j][i] = piece<N>((const T*)a.w + min(n0 + 8 * j, a.n - 1) * a.ldw, k0 + N * i, a.k);
    // (a row past the last repeats it: its values count as the last row's do)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < PIECES; ++i) largest.take(v[j][i]);
    const F8Scale f(block_max<4>(largest.value(), part));
    if (threadIdx.x == 0) a.scales[(int64_t)nb * blocks + kb] = f.scale;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (n0 + 8 * j >= a.n) continue;
        Codes w;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            auto at = [&](int i) { return f.quotient(to_f32(v[j][i / N].v[i % N])); };
            w[q] = f8_codes(at(4 * q), at(4 * q + 1), at(4 * q + 2), at(4 * q + 3));
        }
        __builtin_nontemporal_store(w, (Codes*)(a.codes + (int64_t)(n0 + 8 * j) * blocks * kF8Block + k0));
    }
}

template <class T>
int launch(const QuantizeF8& a, hipStream_t st) {
    const int64_t tiles = f8_padded(a.n) / kF8Block * (f8_padded(a.k) / kF8Block);
    constexpr int threads = 256;
    if (tiles * threads >= kMaxThreads) return fail(SEERA_ERR_INVALID_ARGUMENT, "quantize_weights_f8: the matrix is too large");
    if (a.transposed) hipLaunchKernelGGL((quantize_rows<T>), dim3((uint32_t)tiles), dim3(threads), 0, st, a);
    else hipLaunchKernelGGL((quantize_columns<T>), dim3((uint32_t)tiles), dim3(threads), 0, st, a);
    SEERA_HIP_TRY(hipGetLastError());
    return SEERA_OK;
}

}  // namespace

int quantize_weights_f8(const QuantizeF8& a, hipStream_t st) {
    return a.dtype == SEERA_DTYPE_F32 ? launch<float>(a, st) : a.dtype == SEERA_DTYPE_F16 ? launch<f16_t>(a, st) : launch<bf16_t>(a, st);
}

}  // namespace seera
