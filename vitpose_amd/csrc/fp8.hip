// Products of e4m3 operands with one f32 scale per block of 128:
//
//   y[m][n] = sum_kb  sx[kb][m] sw[n / 128][kb]  sum_{k in block kb} qx[m][k] qw[n][k]   (+ bias, GELU, + residual)
//
// x is cut along K (a scale per row and 128 values), w into 128 x 128 squares; scale = (largest magnitude) / 448, so the
// largest value of a block becomes the largest e4m3 number.  K is padded to a multiple of 128 with zeros.
//
// Sums are f32 with one exception that is the hardware's: an fp8 matrix instruction adds products eight at a time, aligned to
// the largest of the eight with 13 bits kept below its leading one (both the 16x16x32 and the 16x16x128 form; eights meet in
// full f32).  That is 5e-5 of the result's norm on data with a wide spread, against 2e-3 for the bf16 rounding of the result
// and 3e-2 for the rounding of the operands to e4m3.
#include <algorithm>
#include <cmath>

#include "common.h"
#include "vitpose_hip.h"

namespace {

constexpr int BLK = 128;                        // values per scale = reduction steps per K tile = bytes per tile row
constexpr int UNIT = 64 * BLK;                  // 64 rows of one K tile, 8 KiB
constexpr float kTiny = 7.888609052210118e-31f; // 2^-100: a block below it is stored as zeros (448 / amax is finite)

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(4))) int i32x4;

// scale and multiplier of a block from the bit pattern of its largest magnitude (NaN orders above infinity): a block
// with anything that is not finite gets a NaN scale
__device__ __forceinline__ void block_scale(uint32_t bits, float& scale, float& inv) {
    const float amax = __uint_as_float(bits);
    const bool live = amax >= kTiny;
    inv = live ? 1.0f / amax * 448.0f : 0.f;
    scale = live ? amax * (1.0f / 448.0f) : 0.f;
    if (bits >= 0x7F800000u) scale = __uint_as_float(0x7FC00000u);
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// four values as e4m3, nearest, ties to even
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
    const int t = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, t, true);
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    if constexpr (sizeof(T) == 2) {
        const bf16x8 b = *reinterpret_cast<const bf16x8*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)b[i];
    } else {
        const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
    }
}

// ---- rows: sixteen lanes hold a block of one row, a workgroup sixteen rows of DEEP blocks ----
// HBM-bound; all loads of a lane are on their way before the first is used, and the scales of sixteen rows lie next to each other.
// 24576 x 5120 from bf16 60 us = 6.4 TB/s (in a loop by itself 67, blocks dealt out one by one 77).
template <typename T, int DEEP>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* __restrict__ x, long ldx, int M, int K, int KB, int groups,
                                                            long work, uint8_t* __restrict__ q, float* __restrict__ scale) {
    const int sub = threadIdx.x >> 4, l = threadIdx.x & 15;
    for (long w = blockIdx.x; w < work; w += gridDim.x) {
        const long row = w / groups * 16 + sub;
        const int b0 = (int)(w % groups) * DEEP;
        float v[DEEP][8];
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            const int k = (b0 + d) * BLK + l * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[d][i] = 0.f;
            if (row < M && k < K) load8(x + row * ldx + k, v[d]);
        }
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, abs_bits(v[d][i]));
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
            float s, inv;
            block_scale(m, s, inv);
            uint2 out;
            out.x = pack_e4m3(v[d][0] * inv, v[d][1] * inv, v[d][2] * inv, v[d][3] * inv);
            out.y = pack_e4m3(v[d][4] * inv, v[d][5] * inv, v[d][6] * inv, v[d][7] * inv);
            if (row < M && b0 + d < KB) {
                *reinterpret_cast<uint2*>(q + row * ((long)KB * BLK) + (b0 + d) * BLK + l * 8) = out;
                if (l == 0) scale[(long)(b0 + d) * M + row] = s;
            }
        }
    }
}

// ---- rows behind a LayerNorm: a wave holds a row, four blocks of it at a time, and the LayerNorm's weights ----
// Statistics in f32, the variance from differences.  HBM-bound: the next row is on its way while one is rounded; 24576 x 1280 30 us =
// 5.3 TB/s (the LayerNorm to bf16 and the rounding as two launches: 31 + 19).
template <int NB>
__global__ __launch_bounds__(256) void layernorm_rows_kernel(const float* __restrict__ x, const float* __restrict__ gamma,
                                                             const float* __restrict__ beta, float eps, int M, int E, int KB,
                                                             uint8_t* __restrict__ q, float* __restrict__ scale) {
    const int lane = threadIdx.x & 63, wave = blockIdx.x * 4 + (threadIdx.x >> 6), waves = gridDim.x * 4;
    const int k0 = (lane >> 4) * BLK + (lane & 15) * 8;
    float ga[NB][8], be[NB][8], v[NB][8], next[NB][8];
    auto fetch = [&](long row) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
            if (k0 + b * 512 < E) load8(x + row * E + k0 + b * 512, next[b]);
    };
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int i = 0; i < 8; ++i) ga[b][i] = be[b][i] = next[b][i] = 0.f;
        if (k0 + b * 512 < E) {
            load8(gamma + k0 + b * 512, ga[b]);
            load8(beta + k0 + b * 512, be[b]);
        }
    }
    const float n = 1.0f / (float)E;
    if (wave < M) fetch(wave);
    for (long row = wave; row < M; row += waves) {
        float sum = 0.f, sq = 0.f;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 8; ++i) { v[b][i] = next[b][i]; sum += v[b][i]; }
        if (row + waves < M) fetch(row + waves);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
        const float mean = sum * n;
#pragma unroll
        for (int b = 0; b < NB; ++b)
            if (k0 + b * 512 < E)
#pragma unroll
                for (int i = 0; i < 8; ++i) { v[b][i] -= mean; sq += v[b][i] * v[b][i]; }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) sq += __shfl_xor(sq, o, 64);
        const float rstd = rsqrtf(sq * n + eps);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[b][i] = v[b][i] * rstd * ga[b][i] + be[b][i];         // (zeros behind the row's end)
                m = max(m, abs_bits(v[b][i]));
            }
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
            float s, inv;
            block_scale(m, s, inv);
            const int kb = b * 4 + (lane >> 4);
            if (kb < KB) {
                uint2 out;
                out.x = pack_e4m3(v[b][0] * inv, v[b][1] * inv, v[b][2] * inv, v[b][3] * inv);
                out.y = pack_e4m3(v[b][4] * inv, v[b][5] * inv, v[b][6] * inv, v[b][7] * inv);
                *reinterpret_cast<uint2*>(q + row * ((long)KB * BLK) + k0 + b * 512) = out;
                if ((lane & 15) == 0) scale[(long)kb * M + row] = s;
            }
        }
    }
}

// ---- weights: one workgroup per 128 x 128 square, 64 values a thread in registers between the two halves ----
template <typename T>
__global__ __launch_bounds__(256) void quantize_weight_kernel(const T* __restrict__ w, long ldw, int N, int K, int KB,
                                                              uint8_t* __restrict__ q, float* __restrict__ scale) {
    __shared__ uint32_t part[4];
    const int kb = blockIdx.x % KB, nb = blockIdx.x / KB;
    const int r = threadIdx.x >> 4, k = kb * BLK + (threadIdx.x & 15) * 8;
    float v[8][8];
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int n = nb * BLK + j * 16 + r;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] = 0.f;
        if (n < N && k < K) load8(w + (long)n * ldw + k, v[j]);
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, abs_bits(v[j][i]));
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
    __syncthreads();
    m = max(max(part[0], part[1]), max(part[2], part[3]));
    float s, inv;
    block_scale(m, s, inv);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int n = nb * BLK + j * 16 + r;
        if (n >= N) continue;
        uint2 out;
        out.x = pack_e4m3(v[j][0] * inv, v[j][1] * inv, v[j][2] * inv, v[j][3] * inv);
        out.y = pack_e4m3(v[j][4] * inv, v[j][5] * inv, v[j][6] * inv, v[j][7] * inv);
        *reinterpret_cast<uint2*>(q + (long)n * ((long)KB * BLK) + k) = out;
    }
    if (threadIdx.x == 0) scale[(long)nb * KB + kb] = s;
}

struct Args {
    int M, N, KB;
    const uint8_t* xq; long ldx;
    const float* xs;
    const uint8_t* wq; long ldw;
    const float* ws;
    const float* bias;
    int act, out_f32;
    void* out; long ldo;
    const float* resid; long ldr;
    float* oscale;                                            // not NULL: `out` is codes, these are their scales
};

__device__ __forceinline__ void dma16(const void* src, char* lds) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                     (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}

// fragment: 16 rows x 128 bytes; a lane holds 32 consecutive bytes of row li (both operands use the same order of k, so
// which k a byte of a lane stands for does not matter)
__device__ __forceinline__ i32x8 frag(const char* unit, int f, int lane) {
    const int g = lane >> 4, li = lane & 15, r = f * 16 + li;
    const char* u = unit + r * 128;
    const i32x4 lo = *reinterpret_cast<const i32x4*>(u + (((2 * g) ^ (r & 7)) << 4));
    const i32x4 hi = *reinterpret_cast<const i32x4*>(u + (((2 * g + 1) ^ (r & 7)) << 4));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

__device__ __forceinline__ f32x4 mfma_fp8(i32x8 a, i32x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
}

// GELU within a few roundings of ITSELF wherever x lies, because a block's scale makes the largest of 128 results the largest code
// however small they are (an absolute error of 2.5e-5, which 16 bits beside 1 do not show, was a quarter of results near 1e-4 and turned a
// block of zeros into codes of 448).  With t = |x|:  gelu(x) = (x + t) / 2 - h(t),  h(t) = t erfc(t / sqrt 2) / 2 = exp(-t^2 / 2) s P(s),
// s = t / (t + 4.25), P of degree 7 (tools/fit_gelu_poly.py: relative error of the fit 1.2e-7); together within (14 + 3 t + 1.5 t^2) 2^-24.
// Beyond 14.5 h is zero in 32 bits.  NaN enters arithmetically through x.  Measured against a polynomial of absolute error: 24576 x 5120 x
// 1280 to codes 276 us (272), to bf16 248 (243); 12288 rows over K 768 the same.
__device__ __forceinline__ f32x4 gelu(f32x4 v) {
    constexpr float P[8] = {2.696806986e-01f, -1.010334584e+00f, 9.949192922e-01f, 1.487152155e+00f,
                            -5.289770082e+00f, 6.903372525e+00f, -5.080851913e+00f, 2.124999744e+00f};
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const float a = fabsf(v[r]), t = fminf(a, 14.5f), s = t * __builtin_amdgcn_rcpf(t + 4.25f);
        float p = P[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) p = fmaf(p, s, P[i]);
        v[r] = fmaf(0.5f, a, 0.5f * v[r]) - p * s * __builtin_amdgcn_exp2f(t * t * -0.72134752044448170f);
    }
    return v;
}

// Rows of any length: vectors that need only their elements' alignment (the memory takes them: 2585 x 3307 x 496 16 us,
// 30 value by value).
typedef f32x4 f32x4_u __attribute__((aligned(4)));
typedef bf16x4 bf16x4_u __attribute__((aligned(2)));
typedef bf16x8 bf16x8_u __attribute__((aligned(2)));

// four columns j .. j + 3 of a row of the residual (only those below N)
__device__ __forceinline__ f32x4 load_resid(const Args& a, long row, int j) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    const float* p = a.resid + row * a.ldr + j;
    if (j + 3 < a.N) v = *reinterpret_cast<const f32x4_u*>(p);
    else
        for (int r = 0; r < 4; ++r)
            if (j + r < a.N) v[r] = p[r];
    return v;
}

// and of the result
__device__ __forceinline__ void store4(const Args& a, long row, int j, f32x4 v) {
    const bool whole = j + 3 < a.N;
    if (a.out_f32) {
        float* o = (float*)a.out + row * a.ldo + j;
        if (whole) *reinterpret_cast<f32x4_u*>(o) = v;
        else
            for (int r = 0; r < 4; ++r)
                if (j + r < a.N) o[r] = v[r];
    } else {
        bf16* o = (bf16*)a.out + row * a.ldo + j;
        if (whole) *reinterpret_cast<bf16x4_u*>(o) = pack4(v[0], v[1], v[2], v[3]);
        else
            for (int r = 0; r < 4; ++r)
                if (j + r < a.N) o[r] = (bf16)v[r];
    }
}

__device__ __forceinline__ f32x4 finish(const Args& a, f32x4 v, f32x4 bias) {
    v += bias;
    if (a.act) v = gelu(v);
    return v;
}

__device__ __forceinline__ f32x4 load_bias(const Args& a, int j) {
    f32x4 b = {0.f, 0.f, 0.f, 0.f};
    if (a.bias)
        for (int r = 0; r < 4; ++r)
            if (j + r < a.N) b[r] = a.bias[j + r];
    return b;
}

// BM x BN tile, 2 x WN waves of BM / 2 x BN / WN.  128 x 128 tiles are bound by what the CUs take in together, 12.5 TB/s: a K tile
// brings 32 KB for 4.2 MFLOP, one of 256 x 256 64 KB for 16.8, and takes in 8 TB/s; of its 156 us (below) the loads alone take 141, the
// loop without them 128.  LDS is a ring of RING units: behind the K tile being multiplied and the next one, the loads of RING - 2 U more
// units are in flight (with none, the 256 x 256 tile waits for every burst of loads: 2 us a K tile for 0.9 of matrix instructions).
// A lane's accumulators are in f32 units; a K tile's product starts from zero and is added with its block's scale (one FMA
// a value: half of the matrix instructions' time, on another unit).  Measured: 24576 x 1280 x 5120 156 us by itself, 160 behind the
// rounding of its rows = 2.0 PFLOP/s on 256 x 256 tiles, 201 on 128 x 128.
// OUT: what is stored (the dtype tag): one kernel each, or the registers of one epilogue are spilled in another.
template <int BM, int BN, int WN, int RING, int OUT>
__global__ __launch_bounds__(128 * WN, 2) void fp8_kernel(Args a, int tiles_n) {
#ifdef __HIP_DEVICE_COMPILE__   // (the host pass has no buffer resources)
    constexpr int NT = 128 * WN, UX = BM / 64, UY = BN / 64, U = UX + UY, FM = BM / 32, FN = BN / WN / 16;
    constexpr int PER = 512 / NT;                             // sixteen-byte pieces of a unit a thread fetches
    constexpr int XG = 4, PARTS = FM / XG;                    // fragments of x in registers at a time
    constexpr int PITCH = FN * 32 + 16;                       // bytes of a row of a wave's result patch
    static_assert(FM % XG == 0 && PARTS <= 2 && FN * 16 <= 64 && 64 % (FN * 16) == 0, "a wave's columns lie in one unit");
    static_assert(RING >= 2 * U && 2 * WN * 16 * PITCH <= RING * UNIT, "two K tiles, and the patches in their place");
    constexpr int SROWS = BM / (2 * WN), SBYTES = 2 * WN * 256;   // scales: a wave fetches SROWS rows' of a K tile
    static_assert(SROWS <= 64, "one value a lane");
    __shared__ __attribute__((aligned(16))) char lds[RING * UNIT + 2 * SBYTES];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN, g = lane >> 4, li = lane & 15;
    const int work = xcd_remap(blockIdx.x, gridDim.x);
    const int i0 = work / tiles_n * BM, j0 = work % tiles_n * BN;
    const int r0 = tid >> 3, c = ((tid & 7) ^ (r0 & 7)) * 16;
    // Buffer loads: a scalar base and K offset, one 32-bit offset a piece (rows behind the end repeat the last one: they feed
    // what nobody stores), no 64-bit address arithmetic in the loop.
    uint32_t off[U][PER];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int h = 0; h < PER; ++h) {
            const int r = (u < UX ? u : u - UX) * 64 + h * (NT / 8) + r0;
            off[u][h] = u < UX ? min(r, a.M - 1 - i0) * (uint32_t)a.ldx + c : min(r, a.N - 1 - j0) * (uint32_t)a.ldw + c;
        }
    const auto xsrc = __builtin_amdgcn_make_buffer_rsrc((void*)(a.xq + i0 * a.ldx), 0, -1, 0x00020000);
    const auto wsrc = __builtin_amdgcn_make_buffer_rsrc((void*)(a.wq + j0 * a.ldw), 0, -1, 0x00020000);
    auto load = [&](int u, int kb, int slot) {                // unit u of K tile kb (past the end: the last one again)
        char* dst = lds + slot * UNIT + wave * 1024;
        const int k = min(kb, a.KB - 1) * BLK;
#pragma unroll
        for (int h = 0; h < PER; ++h)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(u < UX ? xsrc : wsrc, (__attribute__((address_space(3))) void*)(dst + h * (NT * 16)),
                                                     16, off[u][h], k, 0, 0);
    };
    f32x4 acc[FM][FN];
#pragma unroll
    for (int m = 0; m < FM; ++m)
#pragma unroll
        for (int n = 0; n < FN; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    // (nothing in this launch writes the scales: constant memory, so that a scalar load fetches the wave's)
    const auto sw = (const __attribute__((address_space(4))) float*)(a.ws + (long)min((j0 + wn * FN * 16) / BLK, (a.N - 1) / BLK) * a.KB);
    // The scales of the tile's rows go through LDS as well (two K tiles' worth): fetched into registers they would be waited for
    // together with every load to LDS behind them.
    const uint32_t soff = (uint32_t)min(i0 + wave * SROWS + min(lane, SROWS - 1), a.M - 1) * 4;
    auto scales = [&](int kb) {
        const auto src = __builtin_amdgcn_make_buffer_rsrc((void*)(a.xs + (long)min(kb, a.KB - 1) * a.M), 0, -1, 0x00020000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            src, (__attribute__((address_space(3))) void*)(lds + RING * UNIT + (kb & 1) * SBYTES + wave * 256), 4, soff, 0, 0, 0);
    };
    scales(0);
    float swt = sw[0];
#pragma unroll
    for (int q = 0; q < RING - U; ++q) load(q % U, q / U, q);
    int base = 0;                                             // ring slot of the current K tile's first unit
    auto slot = [&](int u) { const int q = base + u; return q >= RING ? q - RING : q; };
#pragma unroll 1
    for (int t = 0; t < a.KB; ++t) {
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((RING - 2 * U) * PER) : "memory");
        __builtin_amdgcn_s_barrier();                         // K tile t has landed, K tile t - 1 has been read
        asm volatile("" ::: "memory");
        float f[FM];
#pragma unroll
        for (int m = 0; m < FM; ++m) {
            const int r = (wm * FM + m) * 16;
            f[m] = *reinterpret_cast<const float*>(lds + RING * UNIT + (t & 1) * SBYTES + r / SROWS * 256 + (r % SROWS + li) * 4);
        }
        const char* lx0 = lds + slot(wm * (UX / 2)) * UNIT;
        const char* lx1 = lds + slot(wm * (UX / 2) + UX / 2 - 1) * UNIT;
        const char* ly = lds + slot(UX + wn * FN * 16 / 64) * UNIT;
        const int yoff = wn * FN % 4;
        i32x8 xf[XG], yf[2];
        yf[0] = frag(ly, yoff, lane);
#pragma unroll
        for (int m = 0; m < XG; ++m) xf[m] = frag(lx0, m, lane);
        scales(t + 1);
#pragma unroll
        for (int q = RING - U; q < RING; ++q) load(q % U, t + q / U, slot(q));
#pragma unroll
        for (int m = 0; m < FM; ++m) f[m] *= swt;
        swt = sw[min(t + 1, a.KB - 1)];
        __builtin_amdgcn_sched_barrier(0);
        // One matrix instruction, then the four FMAs of the one issued LAG before it: between a matrix instruction and the
        // first use of its result there have to be eleven others, or the compiler fills up with waits.
        constexpr int ALL = PARTS * XG * FN, LAG = 3;
        f32x4 d[LAG + 1];
#pragma unroll
        for (int i = 0; i < ALL + LAG; ++i) {
            const int part = i / (XG * FN), n = i / XG % FN, m = i % XG;
            if (i < ALL) {
                if (m == 0 && i + XG < ALL) yf[(n + 1) & 1] = frag(ly, yoff + (n + 1) % FN, lane);
                d[i % (LAG + 1)] = mfma_fp8(yf[n & 1], xf[m], f32x4{0.f, 0.f, 0.f, 0.f});
                if (PARTS > 1 && part == 0 && n == FN - 1) xf[m] = frag(lx1, m, lane);
            }
            if (i >= LAG) {
                const int j = i - LAG, p = j / (XG * FN) * XG + j % XG, q = j / XG % FN;
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[p][q][r] = fmaf(d[j % (LAG + 1)][r], f[p], acc[p][q][r]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        base = base + U >= RING ? base + U - RING : base + U;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");          // no load may land in LDS that is used for something else
    __syncthreads();
    f32x4 bias[FN];
    const int jw = j0 + wn * FN * 16, iw = i0 + wm * FM * 16;
#pragma unroll
    for (int n = 0; n < FN; ++n) bias[n] = load_bias(a, jw + n * 16 + g * 4);
    if constexpr (OUT == VP_E4M3) {
        // The result as codes: a block of a row lies in PW waves, which meet at its largest magnitude in LDS.
        constexpr int PW = BLK / (FN * 16), ROWS = FM * 16, CPITCH = FN * 16 + 16, SEG = FN;
        static_assert(2 * WN * ROWS * 4 + 2 * WN * 16 * CPITCH <= RING * UNIT, "maxima and patches");
        uint32_t* top = (uint32_t*)lds;
        char* patch = lds + 2 * WN * ROWS * 4 + wave * 16 * CPITCH;
#pragma unroll
        for (int m = 0; m < FM; ++m) {
            uint32_t most = 0;
#pragma unroll
            for (int n = 0; n < FN; ++n) {
                acc[m][n] = finish(a, acc[m][n], bias[n]);
                if (jw + FN * 16 > a.N) {                     // (columns behind the end: padding)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (jw + n * 16 + g * 4 + r >= a.N) acc[m][n][r] = 0.f;
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) most = max(most, abs_bits(acc[m][n][r]));
            }
            most = max(most, (uint32_t)__shfl_xor((int)most, 16, 64));
            most = max(most, (uint32_t)__shfl_xor((int)most, 32, 64));
            if (g == 0) top[wave * ROWS + m * 16 + li] = most;
        }
        __syncthreads();
        const int jb = jw / BLK;
        const bool inside = jb * BLK < a.N;
#pragma unroll
        for (int m = 0; m < FM; ++m) {
            uint32_t most = 0;
#pragma unroll
            for (int p = 0; p < PW; ++p) most = max(most, top[(wave - wn % PW + p) * ROWS + m * 16 + li]);
            float scale, inv;
            block_scale(most, scale, inv);
            const int row = iw + m * 16 + li;
            if (inside && wn % PW == 0 && g == 0 && row < a.M) a.oscale[(long)jb * a.M + row] = scale;
#pragma unroll
            for (int n = 0; n < FN; ++n)
                *reinterpret_cast<uint32_t*>(patch + li * CPITCH + n * 16 + g * 4) =
                    pack_e4m3(acc[m][n][0] * inv, acc[m][n][1] * inv, acc[m][n][2] * inv, acc[m][n][3] * inv);
            if (lane < 16 * SEG) {
                const int r = lane / SEG, c16 = lane % SEG * 16, i = iw + m * 16 + r;
                const i32x4 v = *reinterpret_cast<const i32x4*>(patch + r * CPITCH + c16);
                if (inside && i < a.M) *reinterpret_cast<i32x4*>((uint8_t*)a.out + i * a.ldo + jw + c16) = v;
            }
        }
        return;
    }
    if constexpr (OUT == VP_BF16) {
        // through a patch of LDS of the wave's own, sixteen rows at a time, so that a lane stores sixteen bytes of a row
        constexpr int SEG = FN * 2;
        char* patch = lds + wave * 16 * PITCH;
#pragma unroll
        for (int m = 0; m < FM; ++m) {
#pragma unroll
            for (int n = 0; n < FN; ++n) {
                const f32x4 v = finish(a, acc[m][n], bias[n]);
                *reinterpret_cast<bf16x4*>(patch + li * PITCH + n * 32 + g * 8) = pack4(v[0], v[1], v[2], v[3]);
            }
#pragma unroll
            for (int q = 0; q < SEG / 4; ++q) {
                const int at = q * 64 + lane, r = at / SEG, i = iw + m * 16 + r, j = jw + at % SEG * 8;
                const bf16x8 v = *reinterpret_cast<const bf16x8*>(patch + r * PITCH + at % SEG * 16);
                if (i >= a.M || j >= a.N) continue;
                bf16* o = (bf16*)a.out + i * a.ldo + j;
                if (j + 8 <= a.N) *reinterpret_cast<bf16x8_u*>(o) = v;
                else
                    for (int e = 0; e < a.N - j; ++e) o[e] = v[e];
            }
        }
        return;
    }
    // four rows of the residual are on their way before the first is added
    constexpr int AHEAD = FM < 4 ? FM : 4;
    f32x4 res[AHEAD][FN];
    auto fetch = [&](int m) {
#pragma unroll
        for (int n = 0; n < FN; ++n) {
            const int j = jw + n * 16 + g * 4;
            res[m % AHEAD][n] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (OUT == VP_F32 && a.resid && j < a.N) res[m % AHEAD][n] = load_resid(a, min(iw + m * 16 + li, a.M - 1), j);
        }
    };
#pragma unroll
    for (int m = 0; m < AHEAD; ++m) fetch(m);
#pragma unroll
    for (int m = 0; m < FM; ++m) {
        const int i = iw + m * 16 + li;
#pragma unroll
        for (int n = 0; n < FN; ++n) {
            const int j = jw + n * 16 + g * 4;
            f32x4 v = finish(a, acc[m][n], bias[n]);
            if (OUT == VP_F32 && a.resid) v += res[m % AHEAD][n];
            if (i < a.M && j < a.N) store4(a, i, j, v);
        }
        if (m + AHEAD < FM) fetch(m + AHEAD);
    }
#endif
}

// ---- few rows: what counts is how soon the weights have been read, by how many CUs ----
// A workgroup computes 16 FM rows x 16 FN columns; its eight waves take every eighth block of K straight from memory into
// matrix-instruction operands, and the eight partial tiles are added up in LDS in a fixed order.  Rows in f32 or bf16 are
// rounded to e4m3 on the way (a block of a row lies in four lanes): the same codes and scales as the quantizer's, without
// its launch; every workgroup of a row does it again, which few rows can afford.  Measured: one row, 1280 -> 5120 5.6 us; 192 rows of
// codes, 1024 -> 4096 with a GELU 9.5.
template <typename T, int FM, int FN>
__global__ __launch_bounds__(512, 2) void fp8_narrow_kernel(Args a, const T* __restrict__ x, long ldx, int K, int tiles_n) {
    constexpr int TM = 16 * FM, TN = 16 * FN;
    constexpr bool CODES = sizeof(T) == 1;
    __shared__ __attribute__((aligned(16))) float part[8][TM][TN + 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, li = lane & 15;
    const int work = xcd_remap(blockIdx.x, gridDim.x);
    const int i0 = work / tiles_n * TM, j0 = work % tiles_n * TN;
    const T* px[FM];
    const uint8_t* pw[FN];
    const float* ps[FM];
#pragma unroll
    for (int m = 0; m < FM; ++m) {
        const int row = min(i0 + m * 16 + li, a.M - 1);
        px[m] = x + row * ldx + g * 32;
        ps[m] = CODES ? a.xs + row : nullptr;
    }
#pragma unroll
    for (int n = 0; n < FN; ++n) pw[n] = a.wq + min(j0 + n * 16 + li, a.N - 1) * a.ldw + g * 32;
    const float* sw = a.ws + (long)(j0 / BLK) * a.KB;
    f32x4 acc[FM][FN];
#pragma unroll
    for (int m = 0; m < FM; ++m)
#pragma unroll
        for (int n = 0; n < FN; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
    for (int kb = wave; kb < a.KB; kb += 8) {
        i32x8 wf[FN], xf[FM];
        float f[FM];
#pragma unroll
        for (int n = 0; n < FN; ++n) wf[n] = *reinterpret_cast<const i32x8*>(pw[n] + (long)kb * BLK);
        const float s = sw[kb];
        if constexpr (CODES) {
#pragma unroll
            for (int m = 0; m < FM; ++m) {
                xf[m] = *reinterpret_cast<const i32x8*>(px[m] + (long)kb * BLK);
                f[m] = ps[m][(long)kb * a.M] * s;
            }
        } else {
#pragma unroll
            for (int m = 0; m < FM; ++m) {
                float v[4][8];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int k = kb * BLK + g * 32 + q * 8;
#pragma unroll
                    for (int r = 0; r < 8; ++r) v[q][r] = 0.f;
                    if (k < K) load8(px[m] + (long)kb * BLK + q * 8, v[q]);
                }
                uint32_t top = 0;
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int r = 0; r < 8; ++r) top = max(top, abs_bits(v[q][r]));
                top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
                top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
                float inv;
                block_scale(top, f[m], inv);
                f[m] *= s;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    xf[m][2 * q] = (int)pack_e4m3(v[q][0] * inv, v[q][1] * inv, v[q][2] * inv, v[q][3] * inv);
                    xf[m][2 * q + 1] = (int)pack_e4m3(v[q][4] * inv, v[q][5] * inv, v[q][6] * inv, v[q][7] * inv);
                }
            }
        }
#pragma unroll
        for (int m = 0; m < FM; ++m)
#pragma unroll
            for (int n = 0; n < FN; ++n) {
                const f32x4 d = mfma_fp8(wf[n], xf[m], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[m][n][r] = fmaf(d[r], f[m], acc[m][n][r]);
            }
    }
#pragma unroll
    for (int m = 0; m < FM; ++m)
#pragma unroll
        for (int n = 0; n < FN; ++n) *reinterpret_cast<f32x4*>(&part[wave][m * 16 + li][n * 16 + g * 4]) = acc[m][n];
    __syncthreads();
    for (int q = tid; q < TM * TN / 4; q += 512) {
        const int r = q / (TN / 4), c = q % (TN / 4) * 4, i = i0 + r, j = j0 + c;
        if (i >= a.M || j >= a.N) continue;
        f32x4 v = *reinterpret_cast<const f32x4*>(&part[0][r][c]);
#pragma unroll
        for (int w = 1; w < 8; ++w) v += *reinterpret_cast<const f32x4*>(&part[w][r][c]);
        v = finish(a, v, load_bias(a, j));
        if (a.resid) v += load_resid(a, i, j);
        store4(a, i, j, v);
    }
}

int cdiv(long a, long b) { return (int)((a + b - 1) / b); }
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

extern "C" int vp_quantize_fp8_rows(const void* x, int dtype, long ldx, int M, int K, void* q, float* scale,
                                    hipStream_t stream) {
    VP_CHECK_ARG((dtype == VP_F32 || dtype == VP_BF16) && M >= 0 && K >= 8 && K <= 1 << 30 && K % 8 == 0 && ldx >= K && ldx % 8 == 0);
    if (M == 0) return VP_OK;
    VP_CHECK_ARG(x && q && scale && aligned16(x) && aligned16(q));
    const int KB = cdiv(K, BLK);
    // two blocks a lane where there is work enough for it (us, one / two: 24576 x 5120 74 / 67, 24576 x 1280 21 / 19, 12288 x 768 7.6 /
    // 7.9, 192 x 1024 2.7 / 3.1)
    const long tiles = ((long)M + 15) / 16;
    const bool two = tiles * KB >= 8192;
    const int groups = two ? cdiv(KB, 2) : KB;
    const long work = tiles * groups;
    const unsigned grid = (unsigned)std::min<long>(work, 1 << 20);
    if (dtype == VP_F32)
        hipLaunchKernelGGL((two ? quantize_rows_kernel<float, 2> : quantize_rows_kernel<float, 1>), dim3(grid), dim3(256), 0, stream,
                           (const float*)x, ldx, M, K, KB, groups, work, (uint8_t*)q, scale);
    else
        hipLaunchKernelGGL((two ? quantize_rows_kernel<bf16, 2> : quantize_rows_kernel<bf16, 1>), dim3(grid), dim3(256), 0, stream,
                           (const bf16*)x, ldx, M, K, KB, groups, work, (uint8_t*)q, scale);
    VP_LAUNCH_RET();
}

extern "C" int vp_layernorm_fp8(const float* x, const float* gamma, const float* beta, float eps, int M, int E, void* q,
                                float* scale, hipStream_t stream) {
    VP_CHECK_ARG(M >= 0 && M <= 1 << 29 && E >= 8 && E % 8 == 0 && E <= 2048);
    if (M == 0) return VP_OK;
    VP_CHECK_ARG(x && gamma && beta && q && scale && aligned16(x) && aligned16(gamma) && aligned16(beta) && aligned16(q));
    const int KB = cdiv(E, BLK), grid = std::min(cdiv(M, 4), 2048);
    auto kernel = E <= 512 ? layernorm_rows_kernel<1> : E <= 1024 ? layernorm_rows_kernel<2>
                : E <= 1536 ? layernorm_rows_kernel<3> : layernorm_rows_kernel<4>;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, stream, x, gamma, beta, eps, M, E, KB, (uint8_t*)q, scale);
    VP_LAUNCH_RET();
}

extern "C" int vp_quantize_fp8_weight(const void* w, int dtype, long ldw, int N, int K, void* q, float* scale,
                                      hipStream_t stream) {
    VP_CHECK_ARG((dtype == VP_F32 || dtype == VP_BF16) && N >= 1 && K >= 8 && K <= 1 << 30 && K % 8 == 0 && ldw >= K && ldw % 8 == 0);
    VP_CHECK_ARG(w && q && scale && aligned16(w) && aligned16(q));
    const int KB = cdiv(K, BLK);
    const long grid = (long)KB * cdiv(N, BLK);
    if (!grid_fits(grid, 256)) return VP_ERR_UNSUPPORTED;
    if (dtype == VP_F32)
        hipLaunchKernelGGL(quantize_weight_kernel<float>, dim3((unsigned)grid), dim3(256), 0, stream, (const float*)w, ldw, N,
                           K, KB, (uint8_t*)q, scale);
    else
        hipLaunchKernelGGL(quantize_weight_kernel<bf16>, dim3((unsigned)grid), dim3(256), 0, stream, (const bf16*)w, ldw, N, K,
                           KB, (uint8_t*)q, scale);
    VP_LAUNCH_RET();
}

namespace {

int check_fp8(const vp_fp8_args* g) {
    VP_CHECK_ARG(g && g->M >= 0 && g->M <= 1 << 29 && g->N >= 1 && g->K >= BLK && g->K % BLK == 0 && (g->act == 0 || g->act == 1));
    VP_CHECK_ARG(g->out_dtype == VP_F32 || g->out_dtype == VP_BF16 || g->out_dtype == VP_E4M3);
    if (g->M == 0) return VP_OK;
    VP_CHECK_ARG(g->wq && g->ws && g->out && aligned16(g->wq) && aligned16(g->out));
    VP_CHECK_ARG(g->ldw >= g->K && g->ldo >= g->N && g->ldw % 16 == 0);
    VP_CHECK_ARG(g->out_dtype != VP_E4M3 || (g->oscale && g->ldo % 16 == 0 && g->ldo >= (long)cdiv(g->N, BLK) * BLK));
    VP_CHECK_ARG(!g->resid || (g->out_dtype == VP_F32 && g->ldr >= g->N && aligned16(g->resid)));
    return VP_OK;
}

Args make_args(const vp_fp8_args* g) {
    return Args{g->M, g->N, g->K / BLK, (const uint8_t*)g->xq, g->ldx, g->xs, (const uint8_t*)g->wq, g->ldw, g->ws, g->bias,
                g->act, g->out_dtype == VP_F32, g->out, g->ldo, g->resid, g->ldr, g->out_dtype == VP_E4M3 ? g->oscale : nullptr};
}

template <typename T, int FM, int FN>
int launch_narrow(const vp_fp8_args* g, const T* x, long ldx, int K, hipStream_t stream) {
    const int tn = cdiv(g->N, 16 * FN);
    const long grid = (long)cdiv(g->M, 16 * FM) * tn;
    if (!grid_fits(grid, 512)) return VP_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((fp8_narrow_kernel<T, FM, FN>), dim3((unsigned)grid), dim3(512), 0, stream, make_args(g), x, ldx, K, tn);
    VP_LAUNCH_RET();
}

template <typename T>
int launch_narrow(int shape, const vp_fp8_args* g, const T* x, long ldx, int K, hipStream_t stream) {
    if (shape == 0) return launch_narrow<T, 1, 1>(g, x, ldx, K, stream);
    if (shape == 1) return launch_narrow<T, 1, 2>(g, x, ldx, K, stream);
    if (shape == 2) return launch_narrow<T, 2, 2>(g, x, ldx, K, stream);
    return launch_narrow<T, 2, 4>(g, x, ldx, K, stream);
}

// Which kernel: the one that a simple model of the time, in us, puts first.
//   Few rows: 31 ns per 1000 of K and operand row that a workgroup reads (tile rows + columns; rows that have to be rounded on
//   the way count 2.7 times, in f32 four times), a round of 256 workgroups at a time.  Measured, us at 16 / 192 / 768 / 1536 rows of
//   K 5120, N 1280, rows given as codes: 16 x 16 6.6 / 20 / 69 / 136, 16 x 32 8.9 / 16 / 55 / 102, 32 x 32 9.8 / 12 / 38 / 73, 32 x 64
//   15 / 17 / 30 / 57, 128 x 128 29 / 32 / 33 / 34, 256 x 256 59 / 61 / 63 / 63; K 1000, N 777: 3.3 / 5.2 / 12 / 20, 3.8 / 5.2 / 9.4 /
//   16, 4.0 / 4.5 / 8.4 / 14, 5.1 / 5.7 / 8.6 / 12, 7.9 / 12 / 12 / 13.
//   Tiles: a round of 256 takes a part for its beginning and its stores, more with a GELU or a residual, and a part per K tile; of the
//   128 x 128 tiles two share a CU, so a last round that is not full costs half of what it lacks.  Measured, us, 128 x 128 / 256 x 256: 24576 x 1280 x 5120 201 /
//   160, 24576 x 3840 x 1280 178 / 149, 12288 x 2304 x 768 38 / 37, 6144 x 1024 x 4096 42 / 64; with a GELU 24576 x 5120 x 1280 273 /
//   241, 6144 x 4096 x 1024 50 / 54; with a residual 24576 x 1280 x 5120 229 / 201, 12288 x 768 x 768 29 / 31.
enum { TILE_128 = 4, TILE_256 = 5 };
constexpr int kRows[4] = {16, 16, 32, 32}, kCols[4] = {16, 32, 32, 64};

// (a shape that would need more workgroups than a launch takes: never)
int best_narrow(int M, int N, int K, double row_weight, double further, double& us) {
    int best = 0;
    us = HUGE_VAL;
    for (int s = 0; s < 4; ++s) {
        const long wgs = (long)cdiv(M, kRows[s]) * cdiv(N, kCols[s]);
        const double rounds = (double)((wgs + 255) / 256);
        const double t = rounds * (kRows[s] * row_weight + kCols[s]) * K * 31e-6 + (rounds - 1) * further;
        if (t < us && grid_fits(wgs, 512)) { us = t; best = s; }
    }
    return best;
}

int product_kernel(int M, int N, int K, int act, bool resid, double& us) {
    const int s = best_narrow(M, N, K, 1.0, 0.0, us), kb = cdiv(K, BLK);
    const double tiles = (double)cdiv(M, 128) * cdiv(N, 128) / 256, w128 = std::max(1.25, (tiles + 2 * std::ceil(tiles / 2)) / 2);
    const long w256 = ((long)cdiv(M, 256) * cdiv(N, 256) + 255) / 256;
    double t128 = w128 * (1.7 + 0.63 * kb + 1.2 * act), t256 = w256 * (7.0 + 1.84 * kb + 5.0 * act);
    if (!grid_fits((long)cdiv(M, 128) * cdiv(N, 128), 256)) t128 = HUGE_VAL;
    const double tile = std::min(t128, t256);
    if (us <= tile) return s;
    us = tile;
    if (resid) {                        // (the two tiles add up in one order: a residual does not change the product's bits)
        t128 += 1.5 * w128;
        t256 += 10.0 * w256;
    }
    return t128 <= t256 ? TILE_128 : TILE_256;
}

// The few-rows kernel that rounds its rows itself, or -1: a launch of the quantizer costs about 4 us more, a further round of
// workgroups that begin by rounding 2 us (us, one launch / two: 192 x 4096 x 1024 14.8 / 11.5, 384 x 2304 x 768 13.0 / 10.8,
// 384 x 777 x 1000 7.5 / 8.5, 1 x 5120 x 1280 5.1 / 5.6).
int fused_kernel(int M, int N, int K, int dtype) {
    double fused, split;
    const int s = best_narrow(M, N, K, dtype == VP_F32 ? 4.0 : 2.7, 2.0, fused);
    product_kernel(M, N, K, 0, false, split);
    return fused < HUGE_VAL && fused <= split + 4.0 ? s : -1;
}

template <int BM, int BN, int WN, int RING>
int launch_tile(const vp_fp8_args* g, hipStream_t stream) {
    const int tn = cdiv(g->N, BN);
    const long grid = (long)cdiv(g->M, BM) * tn;
    if (!grid_fits(grid, 128 * WN)) return VP_ERR_UNSUPPORTED;
    auto kernel = g->out_dtype == VP_F32 ? fp8_kernel<BM, BN, WN, RING, VP_F32> : fp8_kernel<BM, BN, WN, RING, VP_BF16>;
    if constexpr (BN == BLK)
        if (g->out_dtype == VP_E4M3) kernel = fp8_kernel<BM, BN, WN, RING, VP_E4M3>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(128 * WN), 0, stream, make_args(g), tn);
    VP_LAUNCH_RET();
}

}  // namespace

extern "C" int vp_gemm_fp8(const vp_fp8_args* g, hipStream_t stream) {
    if (int rc = check_fp8(g)) return rc;
    if (g->M == 0) return VP_OK;
    VP_CHECK_ARG(g->xq && g->xs && aligned16(g->xq) && g->ldx >= g->K && g->ldx % 16 == 0);
    VP_CHECK_ARG(g->ldx <= 1 << 22 && g->ldw <= 1 << 22);       // a tile's rows within 32-bit offsets
    // Codes: 128 x 128 tiles, two of which share a CU: one's largest magnitudes, rounding and GELU, 20 us of a 256 x 256 tile, pass
    // under the other's matrix instructions (6144 x 4096 x 1024: 52 us
    // against 65; 24576 x 5120 x 1280: 277 against 301).
    double us;
    const int which = g->out_dtype == VP_E4M3 ? TILE_128 : product_kernel(g->M, g->N, g->K, g->act, g->resid != nullptr, us);
    if (which < TILE_128) return launch_narrow<uint8_t>(which, g, (const uint8_t*)g->xq, g->ldx, g->K, stream);
    if (which == TILE_256) return launch_tile<256, 256, 4, 18>(g, stream);
    // one workgroup a CU: eight waves; two: four waves each (3000 x 2000 x 3000: 31 us against 34; 192 x 4096 x 1024: 8.5 / 8.1)
    if ((long)cdiv(g->M, 128) * cdiv(g->N, 128) > 256) return launch_tile<128, 128, 2, 9>(g, stream);
    return launch_tile<128, 128, 4, 9>(g, stream);
}

extern "C" int vp_linear_fp8_fused(int M, int N, int K, int dtype) {
    return M >= 1 && N >= 1 && K >= 1 && fused_kernel(M, N, K, dtype) >= 0;
}

extern "C" int vp_linear_fp8(const vp_fp8_args* g, const void* x, int dtype, long ldx, int K, void* xq, float* xs,
                             hipStream_t stream) {
    if (int rc = check_fp8(g)) return rc;
    VP_CHECK_ARG((dtype == VP_F32 || dtype == VP_BF16) && K >= 8 && K % 8 == 0 && cdiv(K, BLK) * BLK == g->K);
    VP_CHECK_ARG(ldx >= K && ldx % 8 == 0 && g->out_dtype != VP_E4M3 && (g->M == 0 || g->ldw <= 1 << 22));
    if (g->M == 0) return VP_OK;
    VP_CHECK_ARG(x && aligned16(x));
    const int shape = fused_kernel(g->M, g->N, K, dtype);
    if (shape >= 0)
        return dtype == VP_F32 ? launch_narrow<float>(shape, g, (const float*)x, ldx, K, stream)
                               : launch_narrow<bf16>(shape, g, (const bf16*)x, ldx, K, stream);
    VP_CHECK_ARG(xq && xs);
    if (int rc = vp_quantize_fp8_rows(x, dtype, ldx, g->M, K, xq, xs, stream)) return rc;
    vp_fp8_args p = *g;
    p.xq = xq;
    p.ldx = g->K;
    p.xs = xs;
    return vp_gemm_fp8(&p, stream);
}
