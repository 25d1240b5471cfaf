// matmul_f8.hip -- products of operands in 8 bits (seera_hip_matmul_f8):
//
//   C[m][n] = sum_b sa[m][b] sw[n / 128][b] sum_{k in block b} A[m][k] W[n][k] + bias[n]
//
// A block of 128 along K begins from zero; its sums are multiplied by the two scales
// and added to fp32 sums. W is the matrix instruction's first operand, so a lane holds
// four values of n of one m: the scale product is one number a lane, and a row of C
// is stored four values at a time. Both operands are permuted alike along K (lanes
// 16 g .. 16 g + 15 hold its 16-byte pieces g and g + 4), which changes no sum of products.
//
// 16-bit results take v_mfma_f32_16x16x128_f8f6f4. It cuts each product below 2^-13 of
// the largest of its group of 8 along K (measured; towards zero), and adds in fp32 from there: less than
// 7 * 2^-13 of the sum of the groups' largest products, and 1.4e-5 of the results of random operands, where
// rounding them to 16 bits is 1.7e-3 or 2e-4. An fp32 result
// is held to fp32's roundings: its codes are widened to fp16, which holds each of them,
// and multiplied by v_mfma_f32_16x16x32_f16, at half the rate (2e-8 of the result).
//
// bf16 results, us: 1 x 4096 x 4096 5.5 (codes of W at a copy's 5 TB/s 3.4, an empty launch
// 3.3), 64 x 12288 x 4096 15.4 (10 + 3.3), 8192 x 12288 x 4096 342 to 364: 2.3 PFLOP/s, where
// a product without scales reaches 3.1. The last is bound by power: the clock falls to 1.65 GHz with
// the matrix cores busy for 0.74 of it. Instructions of 32 x 32 x 64 are no faster (3.9 against
// 4.3 PFLOP/s from registers alone); stores, DMA or scaling left out gave 5 % each.
#include <algorithm>
#include <type_traits>

#include "f8.h"
#include "f8_routes.h"
#include "half_tile.h"
#include "inference.h"
#include "io_types.h"
#include "runtime.h"

namespace seera {
namespace {

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx8 __attribute__((ext_vector_type(8)));

// 128 codes along K of 16 rows, and products of two of them.
struct Codes8 {  // as they are
    intx8 v;
    __device__ __forceinline__ Codes8() {}
    __device__ __forceinline__ explicit Codes8(intx8 c) : v(c) {}
};
struct Codes16 {  // as fp16
    half8 v[4];
    __device__ __forceinline__ Codes16() {}
    __device__ __forceinline__ explicit Codes16(intx8 c) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i], 1.f, false), hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i], 1.f, true);
            v[i / 2][i % 2 * 4] = (half_t)lo[0], v[i / 2][i % 2 * 4 + 1] = (half_t)lo[1];
            v[i / 2][i % 2 * 4 + 2] = (half_t)hi[0], v[i / 2][i % 2 * 4 + 3] = (half_t)hi[1];
        }
    }
};
template <class T>
using Codes = std::conditional_t<sizeof(T) == 4, Codes16, Codes8>;
__device__ __forceinline__ floatx4 products(const Codes8& w, const Codes8& a) {
    const floatx4 zero = {0.f, 0.f, 0.f, 0.f};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, a.v, zero, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ floatx4 products(const Codes16& w, const Codes16& a) {
    floatx4 p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) p = __builtin_amdgcn_mfma_f32_16x16x32_f16(w.v[i], a.v[i], p, 0, 0, 0);
    return p;
}
// Two pieces of 16 codes, 64 apart.
__device__ __forceinline__ intx8 fragment(const uint8_t* at) {
    const intx4 lo = *(const intx4*)at, hi = *(const intx4*)(at + 64);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Four values of a row of C from column n on.
template <class T>
__device__ __forceinline__ void store4(const MatmulF8& g, int m, int n, floatx4 v) {
    T* c = (T*)g.c + (int64_t)m * g.ldc + n;
    if (n + 4 <= g.n) {
        Pack<T, 4> p;
        if (g.bias)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += g.bias[n + i];
#pragma unroll
        for (int i = 0; i < 4; ++i) p.v[i] = from_f32<T>(v[i]);
        __builtin_memcpy(c, &p, sizeof(p));  // at any alignment of T, as one access
        return;
    }
    for (int i = 0; n + i < g.n; ++i) c[i] = from_f32<T>(v[i] + (g.bias ? g.bias[n + i] : 0.f));
}

// Two scales are multiplied with each other first. Where their product overflows, or lies below the
// normal numbers and has lost bits, a block's sums may still give ordinary values (0 among them, which times infinity is
// NaN): there the sums are multiplied by the product of the mantissas, and the exponents added. (With a scale that is
// infinite this comes out the same. A block's sums are below 2^25: a product that rounds to 0 costs less than 2^-125.)
__device__ __forceinline__ bool out_of_range(float s) {
    return __builtin_amdgcn_classf(s, 0x004 | 0x010 | 0x080 | 0x200);  // infinite or subnormal
}
__device__ __forceinline__ floatx4 add_scaled(floatx4 acc, floatx4 p, float sa, float sw) {
    const float s = sa * sw, by = __builtin_amdgcn_frexp_mantf(sa) * __builtin_amdgcn_frexp_mantf(sw);
    const int power = __builtin_amdgcn_frexp_expf(sa) + __builtin_amdgcn_frexp_expf(sw);
    const bool apart = out_of_range(s);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float there = fmaf(p[e], s, acc[e]), here = acc[e] + __builtin_amdgcn_ldexpf(p[e] * by, power);
        acc[e] = apart ? here : there;
    }
    return acc;
}

// Whether any of the products that a lane has noted was out of range: three instructions for two of them, no
// branch and no mask among the matrix instructions, where a comparison each costs 2 to 6 % of the small tiles' time. With
// these, 8192 x 12288 x 4096 is as fast as without them, 64 x 4096 x 4096 9.3 -> 9.7 us, 256 x 4096 x 4096 15.3 -> 13.6 (the
// compiler's order of the LDS reads, not theirs).
struct Noted {
    float most = 0.f;
    uint32_t least = ~0u;  // without the sign, less 1: 0 is above all others
    __device__ __forceinline__ void take(float s) {
        most = fmaxf(most, fabsf(s));
        least = min(least, (__float_as_uint(s) << 1) - 1);
    }
    __device__ __forceinline__ bool apart() const { return __any(most == __builtin_huge_valf() || least < (0x00800000u << 1) - 1); }
};

// The sums of every step-th block from `first` on, of scales whose product may be out of range: the kernels only
// note such products, and their waves come here in the end.
template <class T>
__device__ __forceinline__ floatx4 sums_again(const MatmulF8& g, const uint8_t* a, const uint8_t* w, const float* sa, const float* sw, int first, int step) {
    floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int b = first; b < g.blocks; b += step)
        acc = add_scaled(acc, products(Codes<T>(fragment(w + (int64_t)b * kF8Block)), Codes<T>(fragment(a + (int64_t)b * kF8Block))), sa[b], sw[b]);
    return acc;
}

// Where a lane's operands of a tile of 16 x 16 begin in memory.
struct Operands {
    const uint8_t *a, *w;
    const float *sa, *sw;
    __device__ __forceinline__ Operands(const MatmulF8& g, int m0, int n0, int lane) {
        const int64_t kp = (int64_t)g.blocks * kF8Block;
        // rows past the end repeat the last one: their results are not stored
        const int64_t row = min(m0 + (lane & 15), g.m - 1);
        a = g.a + row * kp + 16 * (lane >> 4);
        w = g.w + min(n0 + (lane & 15), g.n - 1) * kp + 16 * (lane >> 4);
        sa = g.a_scales + row * g.blocks, sw = g.w_scales + (int64_t)(n0 / kF8Block) * g.blocks;
    }
};

// The wave's ROWS x COLS results from (m0, n0) on in this way.
template <class T, int ROWS, int COLS>
__device__ __forceinline__ void results_again(const MatmulF8& g, int m0, int n0) {
    const int lane = threadIdx.x & 63;
#pragma unroll 1
    for (int t = 0; t < ROWS / 16 * (COLS / 16); ++t) {
        const int m = m0 + t % (ROWS / 16) * 16, n = n0 + t / (ROWS / 16) * 16;
        if (m >= g.m || n >= g.n) continue;
        const Operands o(g, m, n, lane);
        const floatx4 acc = sums_again<T>(g, o.a, o.w, o.sa, o.sw, 0, 1);
        if (m + (lane & 15) < g.m) store4<T>(g, m + (lane & 15), n + 4 * (lane >> 4), acc);
    }
}

// ---- few rows: operands from memory to registers ----

// A tile of 16 x 16, with the blocks along K dealt to eight waves, whose sums are joined
// in the waves' order. All of a wave's loads for K up to 4096 are in flight at once: 1 x 4096 x
// 4096 in 5.5 us, and 4.4 with W in the caches from the call before, of which an empty launch is 3.3 (the latter
// with loads a ring of registers ahead: 4.6; 16 waves: 4.7).
constexpr int kSplitWaves = 8;
template <class T>
__global__ __launch_bounds__(64 * kSplitWaves) void matmul_f8_split(MatmulF8 g) {
    __shared__ floatx4 sums[kSplitWaves][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles_n = (g.n + 15) / 16;
    const int n0 = (int)(blockIdx.x % tiles_n) * 16, m0 = (int)(blockIdx.x / tiles_n) * 16;
    const Operands o(g, m0, n0, lane);
    floatx4 acc = {0.f, 0.f, 0.f, 0.f};
    Noted noted;
    for (int b = wave; b < g.blocks; b += kSplitWaves) {
        const Codes<T> cw(fragment(o.w + (int64_t)b * kF8Block)), ca(fragment(o.a + (int64_t)b * kF8Block));
        const float s = o.sa[b] * o.sw[b];
        const floatx4 p = products(cw, ca);
        noted.take(s);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = fmaf(p[e], s, acc[e]);
    }
    if (noted.apart()) acc = sums_again<T>(g, o.a, o.w, o.sa, o.sw, wave, kSplitWaves);
    sums[wave][lane] = acc;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int k = 1; k < kSplitWaves; ++k) acc += sums[k][lane];
    if (m0 + (lane & 15) < g.m) store4<T>(g, m0 + (lane & 15), n0 + 4 * (lane >> 4), acc);
}

template <class T>
int launch_split(const MatmulF8& g, hipStream_t st) {
    const int64_t tiles = (int64_t)((g.n + 15) / 16) * ((g.m + 15) / 16);
    if (tiles * 64 * kSplitWaves >= kMaxThreads) return fail(SEERA_ERR_INVALID_ARGUMENT, "matmul_f8: the product is too large");
    hipLaunchKernelGGL((matmul_f8_split<T>), dim3((uint32_t)tiles), dim3(64 * kSplitWaves), 0, st, g);
    SEERA_HIP_TRY(hipGetLastError());
    return SEERA_OK;
}

// ---- tiles through LDS ----

// 4 bytes per lane as dma16 moves 16.
__device__ __forceinline__ void dma4(dma_rsrc_t r, void* lds, uint32_t voff, uint32_t soff) {
    const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)lds;
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds"
                 :
                 : "s"(at), "v"(voff), "s"(r), "s"(soff)
                 : "memory", "m0");
#pragma clang diagnostic pop
}

// A tile of R rows of 128 codes in LDS, its 16-byte pieces moved within a row so that
// the eight rows that eight lanes read at a time lie in eight places. SPREAD: those
// rows are four of one group of SPREAD rows and four of the next (W), else
// consecutive.
template <int SPREAD>
struct CodeTile {
    static __device__ __forceinline__ int turn(int row) { return SPREAD ? (row & 3) | (row / (SPREAD ? SPREAD : 1) & 1) << 2 : row & 7; }
    // Where a lane's two pieces of a row lie; rows that have the same turn lie a multiple of 128 further.
    static __device__ __forceinline__ int place(int row, int g) { return row * 128 + ((g ^ turn(row)) << 4); }
    static __device__ __forceinline__ intx8 read(const uint8_t* tile, int place) {
        const intx4 lo = *(const intx4*)(tile + place), hi = *(const intx4*)(tile + (place ^ 64));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

// Where a workgroup's rows begin and how many bytes of memory a load may reach from there:
// rows past the matrix lie behind them, and are zeros.
struct Panel {
    const uint8_t* rows;
    const float* scales;
    uint32_t bytes, scale_bytes;
    __device__ __forceinline__ Panel(const uint8_t* codes, const float* s, int first, int last, int most, int first_scale, int scales_there, int blocks)
        : rows(codes + (int64_t)first * blocks * kF8Block),
          scales(s + (int64_t)first_scale * blocks),
          bytes((uint32_t)min(last - first, most) * (uint32_t)blocks * kF8Block),
          scale_bytes((uint32_t)scales_there * (uint32_t)blocks * 4u) {}
};

// Small tiles of BM x BN by four waves for products that larger ones would give too few
// workgroups: what bounds them is how much is on its way from memory, so LDS holds
// STAGES stages of two slices each, all but one of them in flight, and a barrier every two slices
// is all that the waves wait for. BM / 16 or four waves along m, the others along n.
template <class T, int BM, int BN, int STAGES>
__global__ __launch_bounds__(256, 1) void matmul_f8_stream(MatmulF8 g, int tiles_m, int tiles) {
    constexpr int WM = BM >= 64 ? 4 : BM / 16, WN = 4 / WM, MT = BM / WM / 16, NT = BN / WN / 16, KS = 2;
    constexpr int PIECES = (BM + BN) * 8, LOADS_K = (PIECES + 255) / 256, ROWS = BM + BN;
    constexpr int SLICE = LOADS_K * 4096 + 2048, STAGE = KS * SLICE, LOADS = KS * (LOADS_K + 2);
    static_assert(BM <= 128 && BN <= 128 && BM % (16 * WM) == 0 && BN % (16 * WN) == 0 && MT && NT && (STAGES - 2) * LOADS < 64, "shapes of a tile");
    typedef CodeTile<0> Tile;
    extern __shared__ __align__(16) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int id = xcd_order(blockIdx.x, tiles), m0 = id % tiles_m * BM, n0 = id / tiles_m * BN;
    const uint32_t kp = (uint32_t)g.blocks * kF8Block;
    const int wm = wave % WM * (BM / WM), wn = wave / WM * (BN / WN);
    const Panel pa(g.a, g.a_scales, m0, g.m, BM, m0, min(g.m - m0, BM), g.blocks);
    const Panel pw(g.w, g.w_scales, n0, g.n, BN, n0 / kF8Block, 1, g.blocks);
    // a piece of 16 bytes each: rows of A, then of W; whole waves have one of the two
    uint32_t at[LOADS_K];
#pragma unroll
    for (int p = 0; p < LOADS_K; ++p) {
        const int row = (p * 256 + tid) >> 3, r = row < BM ? row : row - BM;
        at[p] = row < ROWS ? (uint32_t)r * kp + (((tid & 7) ^ Tile::turn(row)) << 4) : kBufOOB;
    }
    const uint32_t so = (uint32_t)min(tid, BM - 1) * (uint32_t)g.blocks * 4u;
    auto load = [&](int b, uint8_t* to) {
        const bool there = b < g.blocks;
        const int64_t off = (int64_t)b * kF8Block;
#pragma unroll
        for (int p = 0; p < LOADS_K; ++p) {
            const bool of_a = (p * 256 + wave * 64) / 8 < BM;
            dma16(make_dma_rsrc((of_a ? pa.rows : pw.rows) + off, !there ? 0u : of_a ? pa.bytes : pw.bytes), (half_t*)(to + p * 4096 + wave * 1024), at[p], 0u);
        }
        dma4(make_dma_rsrc(pa.scales + b, there ? pa.scale_bytes : 0u), to + LOADS_K * 4096 + wave * 256, so, 0u);
        dma4(make_dma_rsrc(pw.scales + b, there ? 4u : 0u), to + LOADS_K * 4096 + 1024 + wave * 256, 0u, 0u);
    };
    floatx4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
    const int r = lane & 15, gk = lane >> 4;
    const int a_place = Tile::place(wm + r, gk), w_place = Tile::place(BM + wn + r, gk);

    const int rounds = (g.blocks + KS - 1) / KS;
#pragma unroll
    for (int k = 0; k < (STAGES - 1) * KS; ++k) load(k, smem + k * SLICE);
    int stage = 0;
    Noted noted;
    for (int it = 0; it < rounds; ++it) {
        // this stage has landed, and every wave has read all of the one before, which is filled anew
        wait_vm<(STAGES - 2) * LOADS>();
        lds_barrier();
        const uint8_t* now = smem + stage * STAGE;
        uint8_t* before = smem + (stage == 0 ? STAGES - 1 : stage - 1) * STAGE;
#pragma unroll
        for (int k = 0; k < KS; ++k) load((it + STAGES - 1) * KS + k, before + k * SLICE);
        stage = stage + 1 == STAGES ? 0 : stage + 1;
        intx8 a[KS][MT], w[KS][NT];
        float s[KS][MT];
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            const uint8_t* slice = now + k * SLICE;
            const float* scales = (const float*)(slice + LOADS_K * 4096);
#pragma unroll
            for (int j = 0; j < NT; ++j) w[k][j] = Tile::read(slice + j * 2048, w_place);
#pragma unroll
            for (int i = 0; i < MT; ++i) a[k][i] = Tile::read(slice + i * 2048, a_place);
#pragma unroll
            for (int i = 0; i < MT; ++i) s[k][i] = scales[wm + 16 * i + r];
            const float sw = scales[256 + wave * 64];
#pragma unroll
            for (int i = 0; i < MT; ++i) s[k][i] *= sw;
        }
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            Codes<T> cw[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) cw[j] = Codes<T>(w[k][j]);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const Codes<T> ca(a[k][i]);
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const floatx4 p = products(cw[j], ca);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(p[e], s[k][i], acc[i][j][e]);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < MT; ++i) noted.take(s[k][i]);
    }
    if (noted.apart()) {
        results_again<T, 16 * MT, 16 * NT>(g, m0 + wm, n0 + wn);
    } else {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int m = m0 + wm + 16 * i + r, n = n0 + wn + 16 * j + 4 * gk;
                if (m < g.m) store4<T>(g, m, n, acc[i][j]);
            }
    }
    wait_vm<0>();  // (zeros on their way to LDS that another block may have next)
}

template <class T, int BM, int BN, int STAGES>
int launch_stream(const MatmulF8& g, hipStream_t st) {
    constexpr int lds = STAGES * 2 * (((BM + BN) * 8 + 255) / 256 * 4096 + 2048);
    static_assert(lds <= 160 * 1024, "LDS of a compute unit");
    const int64_t tiles_m = (g.m + BM - 1) / BM, tiles = tiles_m * ((g.n + BN - 1) / BN);
    if (tiles * 256 >= kMaxThreads) return fail(SEERA_ERR_INVALID_ARGUMENT, "matmul_f8: the product is too large");
    auto kern = matmul_f8_stream<T, BM, BN, STAGES>;
    if (lds > 65536)
        SEERA_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    hipLaunchKernelGGL(kern, dim3((uint32_t)tiles), dim3(256), lds, st, g, (int)tiles_m, (int)tiles);
    SEERA_HIP_TRY(hipGetLastError());
    return SEERA_OK;
}

// A tile of BM x BN by WM x WN waves; STAGES stages of LDS, one slice of 128 along K each,
// filled by DMA. In a wave, W's fragments of a slice stay in registers and A's
// pass by: NT products of one, while the sums of the products before it are scaled and
// added. With 16-bit results W's rows are permuted so that a lane holds 8 values next to
// each other of a row of C: 16 bytes, and four lanes 64, as with fp32 without it.
template <class T, int BM, int BN, int WM, int WN, int STAGES>
__global__ __launch_bounds__(64 * WM * WN, 2) void matmul_f8_tiles(MatmulF8 g, int tiles_m, int tiles_n) {
    constexpr int THREADS = 64 * WM * WN, MT = BM / WM / 16, NT = BN / WN / 16;
    constexpr int A_BYTES = BM * 128, W_BYTES = BN * 128, STAGE = A_BYTES + W_BYTES + WM * WN * 256;
    constexpr int A_LOADS = BM * 8 / THREADS, W_LOADS = BN * 8 / THREADS;
    static_assert(BM * 8 % THREADS == 0 && BN * 8 % THREADS == 0 && BM / 64 < WM * WN && BN % 128 == 0 && 128 % (16 * NT) == 0 && NT % 2 == 0 && MT >= 2, "shapes of a tile");
    constexpr int N = 16 / sizeof(T), JJ = N / 4;  // values, and products' rows of 4, in 16 bytes
    typedef CodeTile<0> TA;
    typedef CodeTile<JJ == 1 ? 0 : N> TW;
    extern __shared__ __align__(16) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave % WM * (BM / WM), wn = wave / WM * (BN / WN);
    const uint32_t kp = (uint32_t)g.blocks * kF8Block;
    const int total = tiles_m * tiles_n, slices = max(g.blocks, STAGES + 1);  // (of zeros where there are fewer: loads are STAGES slices ahead)

    // Tile v of this launch's order: the blocks of one XCD walk groups of 4 tile rows column by column.
    struct Tile {
        int m0, n0, live;
    };
    auto tile_of = [&](int v) {
        const int id = xcd_order(min(v, total - 1), total), group = id / (4 * tiles_n), in_group = id - group * 4 * tiles_n, rows = min(tiles_m - group * 4, 4);
        return Tile{(group * 4 + in_group % rows) * BM, in_group / rows * BN, v < total};
    };
    // The stream of slices to load: those of a tile, then the next tile's, so that memory is not
    // waited for between tiles. Rows past the matrix lie outside of the bytes that a load may
    // reach, and are zeros. The scales of A's rows are loaded by the first BM / 64 waves, so that a lane
    // finds its MT ones next to each other, W's by the next wave (the others get zeros).
    const bool a_scales = wave < BM / 64;
    const int scale_row = a_scales ? tid / (16 * MT) * (16 * MT) + tid % MT * 16 + tid % (16 * MT) / MT : lane;
    const uint32_t so = (uint32_t)scale_row * (uint32_t)g.blocks * 4u;
    uint32_t ao[A_LOADS], wo[W_LOADS];
#pragma unroll
    for (int p = 0; p < A_LOADS; ++p) ao[p] = (uint32_t)((p * THREADS + tid) >> 3) * kp + (((tid & 7) ^ TA::turn((p * THREADS + tid) >> 3)) << 4);
#pragma unroll
    for (int p = 0; p < W_LOADS; ++p) wo[p] = (uint32_t)((p * THREADS + tid) >> 3) * kp + (((tid & 7) ^ TW::turn((p * THREADS + tid) >> 3)) << 4);
    struct Stream {
        const uint8_t *a, *w;
        const float* scales;
        uint32_t a_bytes, w_bytes, scale_bytes;
    };
    auto stream_of = [&](const Tile& t) {
        Stream s;
        s.a = g.a + (int64_t)t.m0 * kp, s.w = g.w + (int64_t)t.n0 * kp;
        s.scales = a_scales ? g.a_scales + (int64_t)t.m0 * g.blocks : g.w_scales + (int64_t)(t.n0 / kF8Block) * g.blocks;
        const uint32_t rows_a = min(g.m - t.m0, BM), rows_w = min(g.n - t.n0, BN);
        s.a_bytes = t.live ? rows_a * kp : 0u, s.w_bytes = t.live ? rows_w * kp : 0u;
        s.scale_bytes = t.live && wave <= BM / 64 ? (a_scales ? rows_a : (rows_w + kF8Block - 1) / kF8Block) * (uint32_t)g.blocks * 4u : 0u;
        return s;
    };
    constexpr int LOADS = A_LOADS + W_LOADS + 1;
    int v = blockIdx.x, at = 0;  // the tile that is computed; the slice that is loaded next
    Tile tile = tile_of(v);
    Stream from = stream_of(tile), then = stream_of(tile_of(v + gridDim.x));
    // Load l of a slice; after the last one the stream is a slice further. No branch: the loop
    // below stays one block of code, or its sums are moved to its end.
    auto load = [&](int l, uint8_t* stage) {
        uint8_t* to = stage + wave * 1024;
        if (l < A_LOADS) {
            dma16(make_dma_rsrc(from.a, from.a_bytes), (half_t*)(to + l * THREADS * 16), ao[l < A_LOADS ? l : 0], 0u);
        } else if (l < A_LOADS + W_LOADS) {
            const int p = l < A_LOADS || l >= A_LOADS + W_LOADS ? 0 : l - A_LOADS;
            dma16(make_dma_rsrc(from.w, from.w_bytes), (half_t*)(to + A_BYTES + p * THREADS * 16), wo[p], 0u);
        } else {
            dma4(make_dma_rsrc(from.scales, from.scale_bytes), stage + A_BYTES + W_BYTES + wave * 256, so, 0u);
            // a slice further; the bytes in reach stay: a row past the last begins behind them
            const bool end = ++at == slices;
            at = end ? 0 : at;
            const bool zeros = !end && at >= g.blocks;
            from.a = end ? then.a : from.a + 128;
            from.w = end ? then.w : from.w + 128;
            from.scales = end ? then.scales : from.scales + 1;
            from.a_bytes = end ? then.a_bytes : zeros ? 0u : from.a_bytes;
            from.w_bytes = end ? then.w_bytes : zeros ? 0u : from.w_bytes;
            from.scale_bytes = end ? then.scale_bytes : zeros ? 0u : from.scale_bytes;
        }
    };

    // A slice's products in order: A's fragments one after another, each by all of W's; the last
    // TAIL of A's by one of W's after another, so that W's registers become free one by one.
    // Before these, every wave has read all of the slice: its stage is filled anew, with the
    // slice after the next, while the fragments of the next are read.
    constexpr int TAIL = 3, HEAD = (MT - TAIL) * NT, ALL = MT * NT, RING = 4, AS = TAIL + 1;
    static_assert(MT > TAIL && MT % AS == 0 && HEAD >= RING && TAIL * NT >= LOADS && RING <= 2 * TAIL, "room for the steps' work");
    auto row_of = [](int t) { return t < HEAD ? t / NT : MT - TAIL + (t - HEAD) % TAIL; };
    auto col_of = [](int t) { return t < HEAD ? t % NT : (t - HEAD) / TAIL; };
    floatx4 acc[MT][NT], sums[RING];
    Codes<T> w[NT], a[AS];
    float scale[MT], w_scale, quarter[MT / 4], before[TAIL];  // of this slice; of the last rows in the one before
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < RING; ++i) sums[i] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < TAIL; ++i) before[i] = 0.f;
    const int r = lane & 15, gk = lane >> 4;
    const int a_place = TA::place(wm + r, gk), w_place = TW::place(wn + N * (r >> 2) + (r & 3), gk);
    auto read_a = [&](const uint8_t* stage, int i) { a[i % AS] = Codes<T>(TA::read(stage + i * 2048, a_place)); };
    auto read_w = [&](const uint8_t* stage, int j) { w[j] = Codes<T>(TW::read(stage + A_BYTES + (16 * JJ * (j / JJ) + 4 * (j % JJ)) * 128, w_place)); };
    // (a row's two scales are multiplied when its first sums are added: nothing waits for them here)
    auto read_scales = [&](const uint8_t* stage) {
        const float* s = (const float*)(stage + A_BYTES + W_BYTES);
        __builtin_memcpy(scale, __builtin_assume_aligned(s + wm + r * MT, MT % 4 == 0 ? 16 : 8), sizeof(scale));
        w_scale = s[BM + wn / kF8Block];
        // four lanes have the same rows' scales: each looks at a quarter of them
        __builtin_memcpy(quarter, __builtin_assume_aligned(s + wm + r * MT + gk * (MT / 4), MT), sizeof(quarter));
    };
    auto add = [&](int t, float by) {
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[row_of(t)][col_of(t)][e] = fmaf(sums[t % RING][e], by, acc[row_of(t)][col_of(t)][e]);
    };

#pragma unroll
    for (int k = 0; k < STAGES; ++k)
#pragma unroll
        for (int l = 0; l < LOADS; ++l) load(l, smem + k * STAGE);
    wait_vm<(STAGES - 1) * LOADS>();
    lds_barrier();
    read_a(smem, 0);
#pragma unroll
    for (int j = 0; j < NT; ++j) read_w(smem, j);
    int stage = 0;
    Noted noted;
    for (; v < total; v += gridDim.x) {
        for (int s = 0; s < slices; ++s) {
            uint8_t* now = smem + stage * STAGE;
            stage = stage + 1 == STAGES ? 0 : stage + 1;
            const uint8_t* next = smem + stage * STAGE;
#pragma unroll
            for (int t = 0; t < ALL; ++t) {
                if (t == HEAD) {
                    wait_vm<(STAGES - 2) * LOADS>();
                    lds_barrier();
                }
                if (t >= RING && t - RING < HEAD && (t - RING) % NT == 0) scale[(t - RING) / NT] *= w_scale;
                if (t >= RING && t - RING >= HEAD && t - RING < HEAD + TAIL) scale[row_of(t - RING)] *= w_scale;
                if (t == RING + 1)
#pragma unroll
                    for (int i = 0; i < MT / 4; ++i) noted.take(quarter[i] * w_scale);
                if (t < RING) add(ALL - RING + t, before[row_of(ALL - RING + t) - (MT - TAIL)]);
                else add(t - RING, scale[row_of(t - RING)]);
                __builtin_amdgcn_sched_barrier(0);
                sums[t % RING] = products(w[col_of(t)], a[row_of(t) % AS]);
                __builtin_amdgcn_sched_barrier(0);
                if (t < HEAD) {
                    if (t == 0) read_a(now, 1), read_scales(now);
                    if (t == 1) read_a(now, 2);
                    if (t > 1 && t % NT == NT / 2) read_a(now, t / NT + TAIL);
                } else {
                    const int u = t - HEAD;
                    // (after the last slice of the last tile, of a stage of zeros)
                    if (u == 0) read_a(next, 0);
                    if (u % TAIL == TAIL - 1) read_w(next, u / TAIL);
#pragma unroll
                    for (int l = u * LOADS / (TAIL * NT); l < (u + 1) * LOADS / (TAIL * NT); ++l) load(l, now);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int i = 0; i < TAIL; ++i) before[i] = scale[MT - TAIL + i];
        }
#pragma unroll
        for (int t = ALL - RING; t < ALL; ++t) add(t, before[row_of(t) - (MT - TAIL)]);
        if (noted.apart()) {
            results_again<T, 16 * MT, 16 * NT>(g, tile.m0 + wm, tile.n0 + wn);
            noted = Noted();
        } else {
            typedef uint32_t Bits __attribute__((ext_vector_type(4), aligned(2), may_alias));  // at any alignment of T
            const bool whole = tile.m0 + BM <= g.m && tile.n0 + BN <= g.n;
#pragma unroll
            for (int q = 0; q < NT / JJ; ++q) {
                const int n = tile.n0 + wn + 16 * JJ * q + N * gk;
                float bias[N];
#pragma unroll
                for (int e = 0; e < N; ++e) bias[e] = 0.f;
                if (g.bias) {
                    if (whole) {
                        __builtin_memcpy(bias, g.bias + n, sizeof(bias));
                    } else {
#pragma unroll
                        for (int e = 0; e < N; ++e) bias[e] = g.bias[min(n + e, g.n - 1)];
                    }
                }
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const int m = tile.m0 + wm + 16 * i + r;
                    T* c = (T*)g.c + (int64_t)m * g.ldc + n;
                    Pack<T, N> v;
#pragma unroll
                    for (int e = 0; e < N; ++e) v.v[e] = from_f32<T>(acc[i][q * JJ + e / 4][e % 4] + bias[e]);
                    if (whole || (m < g.m && n + N <= g.n)) {
                        Bits bits;
                        __builtin_memcpy(&bits, &v, 16);
                        __builtin_nontemporal_store(bits, (Bits*)c);
                    } else if (m < g.m) {
#pragma unroll
                        for (int e = 0; e < N; ++e)
                            if (n + e < g.n) c[e] = v.v[e];
                    }
                }
            }
        }
        // the next tile adds these sums, times these scales, before its own: both are 0, as 0 * NaN is none
#pragma unroll
        for (int i = 0; i < RING; ++i) sums[i] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < TAIL; ++i) before[i] = 0.f;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
        // the stream is in the next tile
        tile = tile_of(v + gridDim.x);
        then = stream_of(tile_of(v + 2 * gridDim.x));
    }
    wait_vm<0>();  // (zeros on their way to LDS that another block may have next)
}

template <class T, int BM, int BN, int WM, int WN, int STAGES>
int launch_tiles(const MatmulF8& g, hipStream_t st) {
    constexpr int lds = STAGES * ((BM + BN) * 128 + WM * WN * 256);
    static_assert(lds <= 160 * 1024, "LDS of a compute unit");
    const int tiles_m = (g.m + BM - 1) / BM, tiles_n = (g.n + BN - 1) / BN;
    if ((int64_t)tiles_m * tiles_n >= 1 << 30) return fail(SEERA_ERR_INVALID_ARGUMENT, "matmul_f8: the product is too large");
    auto kern = matmul_f8_tiles<T, BM, BN, WM, WN, STAGES>;
    if (lds > 65536)
        SEERA_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    // as many blocks as run at once
    hipLaunchKernelGGL(kern, dim3((uint32_t)std::min(tiles_m * tiles_n, device_cus())), dim3(64 * WM * WN), lds, st, g, tiles_m, tiles_n);
    SEERA_HIP_TRY(hipGetLastError());
    return SEERA_OK;
}

template <class T>
int launch_t(const MatmulF8& g, hipStream_t st) {
    constexpr bool F32 = sizeof(T) == 4;
    if (!g.blocks) {
        // the bias alone: slices of zeros, for which nothing is read, at any size. (Operands may be null then)
        MatmulF8 zeros = g;
        zeros.a = zeros.w = (const uint8_t*)g.c, zeros.a_scales = zeros.w_scales = (const float*)g.c;
        return launch_tiles<T, 128, 128, 2, 2, 3>(zeros, st);
    }
    // offsets inside a tile are 31 bits
    const bool short_rows = (int64_t)256 * g.blocks * kF8Block < kMaxTileSpanBytes;
    switch (short_rows ? f8_way(F32, g.m, g.n, g.blocks, device_cus()) : kSplit) {
        case kStream16x64: return launch_stream<T, 16, 64, 5>(g, st);
        case kStream32x32: return launch_stream<T, 32, 32, 8>(g, st);
        case kStream32x64: return launch_stream<T, 32, 64, 5>(g, st);
        case kStream64x64: return launch_stream<T, 64, 64, 2>(g, st);
        case kTiles128: return launch_tiles<T, 128, 128, 2, 2, 3>(g, st);
        case kTiles128x256: return launch_tiles<T, 128, 256, 2, 4, 3>(g, st);
        case kTiles256:
            if constexpr (!F32) return launch_tiles<T, 256, 256, 2, 4, 2>(g, st);
        default: return launch_split<T>(g, st);
    }
}

}  // namespace

int matmul_f8(const MatmulF8& g, hipStream_t st) {
    return g.dtype == SEERA_DTYPE_F32 ? launch_t<float>(g, st) : g.dtype == SEERA_DTYPE_F16 ? launch_t<f16_t>(g, st) : launch_t<bf16_t>(g, st);
}

}  // namespace seera
