// AdamW with both moments in 8 bits: e4m3 numbers with one f32 scale per block of 128.
//
//   m' = m + (1 - b1)(g - m)        v' = b2 v + (1 - b2) g^2
//   p' = p (1 - lr wd) - lr / (1 - b1^t) m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// A block keeps  m ~ m_code * m_scale  and  sqrt(v) ~ r_code * r_scale,  scale = (largest magnitude) / 448.
//   * m goes to the nearest e4m3 number: with b1 = 0.9 a step moves it further than half a spacing.
//   * sqrt(v) goes to the lower or the upper neighbour, up with probability (x^2 - lo^2) / (hi^2 - lo^2), so that the
//     EXPECTED v is the exact one.  With b2 = 0.999 a step moves v by 0.1 % while neighbours lie 12 to 25 % apart:
//     rounded to nearest, a code never moves while the block's scale decays under it, and v goes with the scale (a
//     simulated block in which half of the gradients shrink tenfold: the steps of the OTHER half have doubled after
//     2500 iterations; with the rounding used here they stay within 5 %).
//   * a non-zero sqrt(v) never rounds to zero (the smallest code is 2^-9 of a scale): the divisor of an element that is
//     small in its block is too large, never eps.  Only a block whose largest root is under 2^-100 is stored as zeros, and its
//     m with it: no m is left without the divisor that belongs to it.
//   * v itself need not be a 32-bit number: the root is taken of squares scaled by a power of four (gradients of 1e-38 to 1e38).
// The random numbers are a hash of the element's position and of a key that the caller gives for the step: the same
// inputs give the same bits, on every replica.
//
// Memory-bound: 18 bytes a parameter (read 4 p + 4 g + 1 m + 1 r, written 4 p + 2 bf16 copy + 1 + 1) against 30 with
// 32-bit moments.  One workgroup per chunk of 2048 elements, eight per lane: sixteen lanes hold a block, so its two
// maxima are four in-wave exchanges, and all of a lane's loads are in flight before the first is used.  The arithmetic is just
// short enough to stay under the memory time (102 instructions an element, 0.5 % slower than the 90 without the scaling under the
// root; with the library's division and square root, 126, it was 3 to 10 % slower).  Measured: 304 M parameters 1018 us = 5.4 TB/s;
// 90 M 275, with the norm in front 377.
#include "common.h"
#include "vitpose_hip.h"

#pragma clang fp contract(off)   // each product and sum rounds on its own: codes next to a border do not depend on fusion

namespace {

constexpr float kTiny = 7.888609052210118e-31f;       // 2^-100: a block below it is stored as zeros (448 / amax is finite)

// 32-bit finalizer of MurmurHash3 (A. Appleby, public domain): every input bit reaches every output bit
__host__ __device__ __forceinline__ uint32_t mix32(uint32_t h) {
    h ^= h >> 16;
    h *= 0x85EBCA6Bu;
    h ^= h >> 13;
    h *= 0xC2B2AE35u;
    return h ^ (h >> 16);
}

__device__ __forceinline__ uint32_t group16_max(uint32_t v) {
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
        const uint32_t w = (uint32_t)__shfl_xor((int)v, o, 64);
        v = v > w ? v : w;
    }
    return v;
}

// scale and multiplier of a block from the bit pattern of its largest magnitude (bits order like the magnitudes, NaN
// above infinity): a block with anything that is not finite gets a NaN scale, so that it stays visible
__device__ __forceinline__ void block_scale(uint32_t bits, float& scale, float& inv) {
    const float amax = __uint_as_float(bits);
    const bool live = amax >= kTiny;
    inv = live ? 1.0f / amax * 448.0f : 0.f;
    scale = live ? amax * (1.0f / 448.0f) : 0.f;
    if (bits >= 0x7F800000u) scale = __uint_as_float(0x7FC00000u);
}

// the e4m3 code of x in [0, 448], rounded to its lower or upper neighbour, but not to zero unless `zero`; u in [0, 1).  Below
// 2^-6 the spacing stays that of the binade above, so there the neighbours are found 2^-6 further up.
__device__ __forceinline__ uint32_t code_up_or_down(float x, float u, bool zero) {
    x = fminf(x, 448.f);
    const bool sub = x < 0.015625f;
    const float z = sub ? 0.015625f : 0.f;
    const uint32_t cut = __float_as_uint(x + z) & 0xFFF00000u;       // three mantissa bits stay
    const float lo = __uint_as_float(cut) - z, hi = __uint_as_float(cut + 0x100000u) - z, lo2 = lo * lo;
    uint32_t code = (cut >> 20) - (sub ? 968u : 960u);               // exponent bias 127 -> 7
    if (u * (hi * hi - lo2) < x * x - lo2) ++code;
    code = code > 126u ? 126u : (code < 1u ? 1u : code);
    return zero ? 0u : code;
}

// sqrt(b2 r^2 + (1 - b2) g^2), the root rounded to nearest but for one value in some four million: a Newton step on v rsq(v).  Both
// numbers are scaled by the power of two that brings the larger one to 1 (its exponent kept within what has a reciprocal), which
// changes no bit of the result: nothing overflows or underflows that the result does not.
__device__ __forceinline__ float new_root(float r, float g, float beta2, float omb2) {
    const uint32_t top = __float_as_uint(fmaxf(fabsf(r), fabsf(g))) & 0x7F800000u;
    const uint32_t e = top < 0x00800000u ? 0x00800000u : (top > 0x7E800000u ? 0x7E800000u : top);
    const float scale = __uint_as_float(0x7F000000u - e);
    r *= scale;
    g *= scale;
    const float v = beta2 * (r * r) + (omb2 * g) * g;
    const float y = v < 1.17549435e-38f ? 0.f : __builtin_amdgcn_rsqf(v);
    const float s = v * y;
    return __builtin_fmaf(__builtin_fmaf(-s, s, v), 0.5f * y, s) * __uint_as_float(e);
}

__global__ __launch_bounds__(256) void adamw8_kernel(
    float* __restrict__ p, const float* __restrict__ g, uint8_t* __restrict__ m8, float* __restrict__ ms,
    uint8_t* __restrict__ r8, float* __restrict__ rs, bf16* __restrict__ half, const long* __restrict__ chunk_start,
    const int* __restrict__ chunk_len, const float* __restrict__ chunk_lr_scale, const float* __restrict__ chunk_wd,
    const long* __restrict__ chunk_state, long numel, long state_numel, float lr, float omb1, float beta2, float omb2,
    float eps, float bc1, float inv_bc2, const double* __restrict__ partials, int npartials, float max_norm,
    float grad_scale, uint32_t key) {
    __shared__ double wave_part[4];
    const int tid = threadIdx.x, i = tid * 8;
    const long s0 = chunk_start[blockIdx.x], q0 = chunk_state[blockIdx.x];
    const int len = chunk_len[blockIdx.x];
    // a row of the table that does not fit the buffers is left out (uniform over the workgroup; by differences, which stay in 64 bits)
    if (len <= 0 || len > 2048 || (len & 3) || (s0 & 3) || (q0 & 127) || s0 < 0 || q0 < 0 || s0 > numel - len ||
        q0 > state_numel - ((len + 127) & ~127))
        return;
    const bool on = i < len, two = i + 4 < len;
    const long o = s0 + (on ? i : 0), o2 = two ? o + 4 : o, q = q0 + (on ? i : 0);
    const f32x4 z = {0.f, 0.f, 0.f, 0.f};
    f32x4 pv[2], gv[2];
    pv[0] = *reinterpret_cast<const f32x4*>(p + o);
    pv[1] = *reinterpret_cast<const f32x4*>(p + o2);
    gv[0] = *reinterpret_cast<const f32x4*>(g + o);
    gv[1] = *reinterpret_cast<const f32x4*>(g + o2);
    const uint2 mc = *reinterpret_cast<const uint2*>(m8 + q), rc = *reinterpret_cast<const uint2*>(r8 + q);
    const float msc = ms[q >> 7], rsc = rs[q >> 7];
    float clip = grad_scale;
    if (npartials > 0) {          // every workgroup adds the same numbers in the same order
        double d = tid < npartials ? partials[tid] : 0.0;
#pragma unroll
        for (int k = 32; k > 0; k >>= 1) d += __shfl_xor(d, k, 64);
        if ((tid & 63) == 0) wave_part[tid >> 6] = d;
        __syncthreads();
        const float tn = (float)sqrt((wave_part[0] + wave_part[1]) + (wave_part[2] + wave_part[3])) * grad_scale;
        clip *= fminf(max_norm / (tn + 1e-6f), 1.f);
        if (tn != tn) clip = tn;  // fminf drops a NaN
    }
    uint32_t mw[2] = {mc.x, mc.y}, rw[2] = {rc.x, rc.y};
    if (len < 2048) {             // (uniform) what lies behind the chunk's end counts as zeros
        if (!on) { gv[0] = z; pv[0] = z; mw[0] = 0; rw[0] = 0; }
        if (!two) { gv[1] = z; pv[1] = z; mw[1] = 0; rw[1] = 0; }
    }
    const float lr_c = lr * chunk_lr_scale[blockIdx.x];
    const float keep = 1.f - lr_c * chunk_wd[blockIdx.x], rate = lr_c / bc1;
    float m[8], r[8];
    uint32_t mmax = 0, rmax = 0;
#pragma unroll
    for (int h = 0; h < 4; ++h) {
        const auto m2 = (h & 1) ? __builtin_amdgcn_cvt_pk_f32_fp8((int)mw[h >> 1], true) : __builtin_amdgcn_cvt_pk_f32_fp8((int)mw[h >> 1], false);
        const auto r2 = (h & 1) ? __builtin_amdgcn_cvt_pk_f32_fp8((int)rw[h >> 1], true) : __builtin_amdgcn_cvt_pk_f32_fp8((int)rw[h >> 1], false);
#pragma unroll
        for (int l = 0; l < 2; ++l) {
            const int k = 2 * h + l;
            const float mk = m2[l] * msc, rk = r2[l] * rsc;
            const float gk = gv[k >> 2][k & 3] * clip, pk = pv[k >> 2][k & 3];
            m[k] = mk + omb1 * (gk - mk);
            r[k] = new_root(rk, gk, beta2, omb2);
            pv[k >> 2][k & 3] = pk * keep - (rate * m[k]) * __builtin_amdgcn_rcpf(r[k] * inv_bc2 + eps);
            const uint32_t mb = __float_as_uint(m[k]) & 0x7FFFFFFFu, rb = __float_as_uint(r[k]) & 0x7FFFFFFFu;
            mmax = mmax > mb ? mmax : mb;
            rmax = rmax > rb ? rmax : rb;
        }
    }
    mmax = group16_max(mmax);
    rmax = group16_max(rmax);
    float mscale, minv, rscale, rinv;
    block_scale(mmax, mscale, minv);
    block_scale(rmax, rscale, rinv);
    const float least = rinv > 0.f ? 0.f : __builtin_inff();      // roots above it have a code
    if (rscale == 0.f) mscale = minv = 0.f;
    uint32_t rcode[2] = {0, 0};
    const uint32_t pos = (uint32_t)(unsigned long)q;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float u = (float)(mix32((pos + k) ^ key) >> 8) * 5.9604644775390625e-8f;
        rcode[k >> 2] |= code_up_or_down(r[k] * rinv, u, !(r[k] > least)) << (8 * (k & 3));
    }
    uint2 mo;
    int t = __builtin_amdgcn_cvt_pk_fp8_f32(m[0] * minv, m[1] * minv, 0, false);
    mo.x = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(m[2] * minv, m[3] * minv, t, true);
    t = __builtin_amdgcn_cvt_pk_fp8_f32(m[4] * minv, m[5] * minv, 0, false);
    mo.y = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(m[6] * minv, m[7] * minv, t, true);
    if (!on) return;
    *reinterpret_cast<f32x4*>(p + o) = pv[0];
    if (two) *reinterpret_cast<f32x4*>(p + o2) = pv[1];
    if (half) {
        *reinterpret_cast<bf16x4*>(half + o) = pack4(pv[0][0], pv[0][1], pv[0][2], pv[0][3]);
        if (two) *reinterpret_cast<bf16x4*>(half + o2) = pack4(pv[1][0], pv[1][1], pv[1][2], pv[1][3]);
    }
    *reinterpret_cast<uint2*>(m8 + q) = mo;
    *reinterpret_cast<uint2*>(r8 + q) = make_uint2(rcode[0], rcode[1]);
    if ((tid & 15) == 0) {
        ms[q >> 7] = mscale;
        rs[q >> 7] = rscale;
    }
}

// sum of squares over a table's chunks in 64 bits, one partial sum per workgroup: workgroup b takes the chunks b,
// b + gridDim.x, ... in order, so the sum depends on the table alone
__global__ __launch_bounds__(1024) void sumsq_chunks_f64_kernel(const float* __restrict__ x, const long* __restrict__ start,
                                                                const int* __restrict__ length, int nchunks, long numel,
                                                                double* __restrict__ partials) {
    __shared__ double part[16];
    const int sub = threadIdx.x >> 8, lane = threadIdx.x & 255;      // four chunks at a time
    double d0 = 0.0, d1 = 0.0;
    // chunks in flight (90 M elements that no cache holds: one 65 us, two 60 = 6.0 TB/s, four 62, eight 63; 100 right behind a step's writes)
    constexpr int DEEP = 2;
    const long stride = (long)gridDim.x * 4;
    for (long c0 = (long)blockIdx.x * 4 + sub; c0 < nchunks; c0 += stride * DEEP) {
        long st[DEEP];
        int len[DEEP];
        f32x4 v[DEEP][2];
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            const long c = c0 + d * stride;
            st[d] = 0;
            len[d] = 0;
            if (c < nchunks) { st[d] = start[c]; len[d] = length[c]; }
        }
        const int i = lane * 4;
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            const bool ok = len[d] > 0 && len[d] <= 2048 && !(len[d] & 3) && !(st[d] & 3) && st[d] >= 0 && st[d] <= numel - len[d];
            v[d][0] = v[d][1] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (ok && i < len[d]) v[d][0] = *reinterpret_cast<const f32x4*>(x + st[d] + i);
            if (ok && i + 1024 < len[d]) v[d][1] = *reinterpret_cast<const f32x4*>(x + st[d] + 1024 + i);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int d = 0; d < DEEP; ++d)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                d0 += (double)v[d][0][k] * v[d][0][k];
                d1 += (double)v[d][1][k] * v[d][1][k];
            }
    }
    d0 += d1;
#pragma unroll
    for (int k = 32; k > 0; k >>= 1) d0 += __shfl_xor(d0, k, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = d0;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int k = 0; k < 16; ++k) t += part[k];
        partials[blockIdx.x] = t;
    }
}

}  // namespace

extern "C" int vp_sumsq_chunks_f64(const float* x, const long* chunk_start, const int* chunk_len, int nchunks,
                                   long numel, double* partials, int npartials, hipStream_t stream) {
    VP_CHECK_ARG(nchunks >= 0 && numel >= 0 && npartials >= 1 && npartials <= 256 && partials);
    VP_CHECK_ARG(nchunks == 0 || (x && chunk_start && chunk_len && ((uintptr_t)x & 15) == 0));
    hipLaunchKernelGGL(sumsq_chunks_f64_kernel, dim3(npartials), dim3(1024), 0, stream, x, chunk_start, chunk_len, nchunks,
                       numel, partials);
    VP_LAUNCH_RET();
}

extern "C" int vp_adamw8_step(float* p, const float* g, void* m_e4m3, float* m_scale, void* r_e4m3, float* r_scale,
                              void* p_bf16, const long* chunk_start, const int* chunk_len, const float* chunk_lr_scale,
                              const float* chunk_wd, const long* chunk_state, int nchunks, long numel, long state_numel,
                              double lr, double beta1, double beta2, double eps, long step, const double* norm_partials,
                              int npartials, float max_norm, float grad_scale, unsigned noise, hipStream_t stream) {
    VP_CHECK_ARG(nchunks >= 0 && step > 0 && numel >= 0 && numel % 4 == 0 && state_numel >= 0 && state_numel % 128 == 0);
    VP_CHECK_ARG(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && (eps == 0 || (eps > 0 && (float)eps >= 1.17549435e-38f)));
    VP_CHECK_ARG(npartials >= 0 && npartials <= 256 && (npartials == 0 || (norm_partials && max_norm > 0.f)));
    if (nchunks == 0) return VP_OK;
    VP_CHECK_ARG(p && g && m_e4m3 && m_scale && r_e4m3 && r_scale && chunk_start && chunk_len && chunk_lr_scale &&
                 chunk_wd && chunk_state);
    VP_CHECK_ARG((((uintptr_t)p | (uintptr_t)g) & 15) == 0 && (((uintptr_t)m_e4m3 | (uintptr_t)r_e4m3 | (uintptr_t)p_bf16) & 7) == 0);
    // eps 0: the smallest normal number in its place, which no root of a live block notices (0 / 0 is no update)
    const float least = eps > 0 ? (float)eps : 1.17549435e-38f;
    const float bc1 = (float)(1.0 - pow(beta1, (double)step)), inv_bc2 = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)step)));
    hipLaunchKernelGGL(adamw8_kernel, dim3(nchunks), dim3(256), 0, stream, p, g, (uint8_t*)m_e4m3, m_scale,
                       (uint8_t*)r_e4m3, r_scale, (bf16*)p_bf16, chunk_start, chunk_len, chunk_lr_scale, chunk_wd,
                       chunk_state, numel, state_numel, (float)lr, (float)(1.0 - beta1), (float)beta2,
                       (float)(1.0 - beta2), least, bc1, inv_bc2, norm_partials, npartials, max_norm, grad_scale, noise);
    VP_LAUNCH_RET();
}
