// Products of rows with the weight of the expert each row belongs to (a mixture-of-experts Linear), ragged:
//
//   y[t]  = x[t] W[e(t)]^T + b[e(t)]          forward            W [E][N][K], b [E][N]
//   dx[t] = dy[t] W[e(t)]                     gradient of x
//   dW[e] = sum_{t: e(t) = e} dy[t]^T x[t]    gradient of W      db[e] = sum_{t: e(t) = e} dy[t]
//
// The rows of expert e are offsets[e] .. offsets[e + 1] of a list; entry i of the list is row rows[i] of the arrays (or
// row i itself without a list), so operands are read, and results written, where they lie: the loader takes a pointer per
// row anyway.  Offsets and list live on the device and are read there: nothing waits for the host.
//
// All three are one tile product C[i][j] = sum_k X[i][k] Y[j][k] with different roles:
//   forward  i = rows, j = N, k = K       X = x (k-contiguous),  Y = W[e] (k-contiguous)
//   dx       i = rows, j = K, k = N       X = dy (k-contiguous), Y = W[e] (k-major: stored P[k][j])
//   dW       i = N,    j = K, k = rows    X = dy (k-major),      Y = x (k-major)
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "vitpose_hip.h"

namespace {

constexpr int BK = 64, UNIT = 64 * BK * 2, THREADS = 512;   // a unit: 64 rows (or columns) x 64 reduction steps, 8 KiB

// sixteen bytes of zeros: what a lane fetches for reduction steps beyond the end (0 x 0: a neighbour's NaN cannot enter)
__device__ __constant__ static const float kZeros[4] = {0.f, 0.f, 0.f, 0.f};

struct Args {
    const int* offsets;
    const int* rows;
    int T, E, N, K;
    const bf16* x; long ldx;        // row operand of the forward product (or x of dW)
    const bf16* w; long ldw, stride_w;
    const float* bias; long stride_b;
    const bf16* dy; long ldy;
    void* out; long ldo;
    float* dw; float* db;
    int zero_rest, slices;
};

struct Span { int lo, hi; };

// inclusive sum over the lanes of a wave: within rows of sixteen, then the rows' last lanes handed on
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);   // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);   // row_shr:2
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);   // row_shr:4
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);   // row_shr:8
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);   // row_bcast:15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);   // row_bcast:31 into rows 2 and 3
    return v;
}

// rows of expert e in the list, kept inside it whatever the offsets say
__device__ __forceinline__ Span span_of(const int* offsets, int e, int T) {
    int lo = offsets[e], hi = offsets[e + 1];
    lo = lo < 0 ? 0 : (lo > T ? T : lo);
    hi = hi < lo ? lo : (hi > T ? T : hi);
    return Span{lo, hi};
}

// What workgroup blockIdx.x of a launch over row tiles (bm list entries each, `per` workgroups a tile) has to do: the
// expert whose rows its tile holds (E: rows behind the last expert or before the first, -1: nothing), the tile's first and last
// list entry and the workgroup's number within the tile.  Every wave scans the experts' tile counts, 64 at a time.  The tiles there ARE are
// dealt out to the XCDs in contiguous runs (the grid is an upper bound: dealing IT out would give seven XCDs more workgroups
// than they have CUs and the eighth next to none; 240 of 275 workgroups: 46 us against 30).
__device__ __forceinline__ int find_tile(const Args& a, int bm, int per, int lane, int& lo, int& hi, int& inner) {
    int total = 0, sum = 0, n = 0;
    Span s{0, 0};
    for (int e0 = 0; e0 < a.E; e0 += 64) {
        const int e = e0 + lane;
        s = Span{0, 0};
        if (e < a.E) s = span_of(a.offsets, e, a.T);
        n = (s.hi - s.lo + bm - 1) / bm;
        sum = wave_scan(n);
        total += __builtin_amdgcn_readlane(sum, 63);
    }
    int begin = 0, end = a.T;                              // entries before begin and from end on are no expert's
    if (a.zero_rest) {
        begin = a.offsets[0];
        end = a.offsets[a.E];
        begin = begin < 0 ? 0 : (begin > a.T ? a.T : begin);
        end = end < 0 ? 0 : (end > a.T ? a.T : end);
    }
    const int rest = (a.T - end + bm - 1) / bm, head = (begin + bm - 1) / bm, groups = (total + rest + head) * per;
    if ((int)blockIdx.x >= groups) return -1;
    const int work = xcd_remap(blockIdx.x, groups), tile = work / per;
    inner = work - tile * per;
    if (tile >= total) {
        const bool behind = tile - total < rest;
        lo = behind ? end + (tile - total) * bm : (tile - total - rest) * bm;
        hi = min(behind ? a.T : begin, lo + bm);
        return a.E;
    }
    int before = 0;
    for (int e0 = 0; e0 < a.E; e0 += 64) {
        if (a.E > 64) {
            const int e = e0 + lane;
            s = Span{0, 0};
            if (e < a.E) s = span_of(a.offsets, e, a.T);
            n = (s.hi - s.lo + bm - 1) / bm;
            sum = wave_scan(n);
        }
        const unsigned long long past = __ballot(before + sum > tile);
        if (past) {
            const int src = __builtin_ctzll(past);
            const int first = __builtin_amdgcn_readlane(before + sum - n, src);
            lo = __builtin_amdgcn_readlane(s.lo, src) + (tile - first) * bm;
            hi = min(__builtin_amdgcn_readlane(s.hi, src), lo + bm);
            return e0 + src;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    return -1;
}

// The expert with the rank-th most rows (equal ones by number); beyond 64 experts the order is theirs.
__device__ __forceinline__ int expert_by_size(const Args& a, int rank, int lane) {
    if (a.E > 64) return rank;
    Span s{0, 0};
    if (lane < a.E) s = span_of(a.offsets, lane, a.T);
    const int n = lane < a.E ? s.hi - s.lo : -1;
    int mine = 0;
    for (int j = 0; j < a.E; ++j) {
        const int other = __builtin_amdgcn_readlane(n, j);
        mine += other > n || (other == n && j < lane);
    }
    return __builtin_ctzll(__ballot(mine == rank && lane < a.E));
}

__device__ __forceinline__ int kmaj_key(int kr) { return ((kr >> 1) & 1) | (((kr >> 3) & 1) << 1); }

// a value in global memory at an address that was picked among several (said in so many words: the compiler no longer
// sees that it is global, and flat instructions wait for LDS too)
template <typename T>
__device__ __forceinline__ T load_at(uintptr_t p) { return *(const __attribute__((address_space(1))) T*)p; }
template <typename T>
__device__ __forceinline__ void store_at(uintptr_t p, T v) { *(__attribute__((address_space(1))) T*)p = v; }

__device__ __forceinline__ void dma16(const void* src, char* lds) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                     (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}

// fragment (16 rows / columns, 32 reduction steps) `f` of an operand tile made of 64-wide units
template <bool KMAJ>
__device__ __forceinline__ bf16x8 frag(const char* tile, int f, int s, int lane) {
    const int g = lane >> 4, li = lane & 15;
    const char* u = tile + (f >> 2) * UNIT;
    if constexpr (!KMAJ) {
        const int r = (f & 3) * 16 + li;
        return *reinterpret_cast<const bf16x8*>(u + r * 128 + ((((s << 2) + g) ^ (r & 7)) << 4));
    } else {
        const int q = li >> 2, p = li & 3, kq = 8 * g + q;
        const char* base = u + s * 4096 + kq * 128 + (((f & 3) ^ kmaj_key(kq)) << 5) + (p << 3);
        const bf16x4 lo = lds_read_tr_raw(base, 0), hi = lds_read_tr_raw(base, 512);
        return cat8(lo, hi);
    }
}

enum { FWD = 0, DX = 1, DW = 2 };

template <int N_>
__device__ __forceinline__ void wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N_) : "memory");
}


// BM x BN tile by eight waves: waves 0-3 (2 x 2 blocks of BM / 2 x BN / 2) take the first 32 reduction steps of every K tile,
// waves 4-7 the other 32, so a CU has two waves per SIMD on blocks as large as four would have; the halves meet through LDS
// once at the end.  S stages: while K tile t is multiplied, the loads of t + 1 .. t + S - 1 are in flight (with two stages the
// 128 x 128 tile needed 1 us per K tile for 0.2 us of matrix instructions).  One barrier per K tile.  Loads past the end fetch
// zeros, so that the counted waits hold.  PER_CU workgroups share a CU.
// What bounds it is what a CU takes in, 51 KB a microsecond from memory and 60 from caches, whatever the depth and however many
// CUs are at it: without its LDS reads and matrix instructions the loop takes 40 us instead of 41.  Measured, inputs in memory:
// forward 12288 x 256 x 4096 47 us = 545 TFLOP/s; 6144 rows of 320 x 5120: forward 43, dW 44 us (39 MB written).
template <int WHAT, int BM, int BN, int S, int PER_CU = 1>
__global__ __launch_bounds__(THREADS, 2 * PER_CU) void grouped_kernel(Args a, int tiles_j, int tiles_i) {
    constexpr bool XK = WHAT == DW, YK = WHAT != FWD;
    constexpr int UX = BM / 64, UY = BN / 64, U = UX + UY, FM = BM / 32, FN = BN / 32, FH = FM / 2, STAGE = U * UNIT;
    constexpr int SWAP = 8 * FH * FN * 1024, PITCH = BN + 16, PATCH = 16 * FH * PITCH;
    constexpr int BYTES = S * STAGE > SWAP ? S * STAGE : SWAP;
    constexpr int LIST = 2048 / PER_CU;                    // entries of the row list that a dW workgroup keeps in LDS at a time
    static_assert(8 * PATCH <= BYTES, "the result patches reuse the stages");
    __shared__ __attribute__((aligned(16))) char lds[BYTES];
    __shared__ int list[XK ? LIST : 1];
    __shared__ float sums_half[XK ? 8 * FM * 16 : 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kg = wave >> 2, wm = (wave >> 1) & 1, wn = wave & 1, g = lane >> 4, li = lane & 15;
    int e, lo, hi, i0 = 0, j0, k_end, kt0 = 0, kt1, slice = 0;
    if constexpr (WHAT == DW) {
        // The tiles that read one panel of x (all of N, one tile of K) run next to each other on one XCD; panels are dealt
        // out to the XCDs in turn, those of the expert with the most rows first: a contiguous eighth of the list each would
        // leave the longest sums to one XCD (6144 rows in shares from 41 to 7 %, 320 x 5120, 128 x 128 tiles: 82 us against 47)
        const int at = blockIdx.x >> 3, panel = at / tiles_i * 8 + (blockIdx.x & 7), per = tiles_j * a.slices;
        if (panel >= a.E * per) return;
        e = expert_by_size(a, panel / per, lane);
        slice = panel % a.slices;
        i0 = at % tiles_i * BM;
        j0 = panel % per / a.slices * BN;
        const Span s = span_of(a.offsets, e, a.T);
        lo = s.lo;
        hi = s.hi;
        k_end = hi - lo;
        const int nk_all = (k_end + BK - 1) / BK, each = (nk_all + a.slices - 1) / a.slices;
        kt0 = min(slice * each, nk_all);
        kt1 = min(kt0 + each, nk_all);
    } else {
        e = find_tile(a, BM, tiles_j, lane, lo, hi, j0);
        if (e < 0) return;
        j0 *= BN;
        k_end = e == a.E ? 0 : (WHAT == FWD ? a.K : a.N);
        kt1 = (k_end + BK - 1) / BK;
    }
    const int NJ = WHAT == FWD ? a.N : a.K;

    f32x4 acc[FM][FN];
#pragma unroll
    for (int m = 0; m < FM; ++m)
#pragma unroll
        for (int n = 0; n < FN; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    f32x4 rs[FM];
#pragma unroll
    for (int m = 0; m < FM; ++m) rs[m] = f32x4{0.f, 0.f, 0.f, 0.f};
    const bool sums = WHAT == DW && a.db && j0 == 0 && wn == 0;

    // a lane's place in a unit: row (or reduction step) r0, sixteen bytes at column cc (k-contiguous) or ck (k-major)
    const int r0 = tid >> 3;
    const int cc = ((tid & 7) ^ (r0 & 7)) * 8;
    const int ck = ((((tid & 7) >> 1) ^ kmaj_key(r0)) * 2 + (tid & 1)) * 8;
    const bf16* px[UX];
    const bf16* py[UY];
    if constexpr (!XK) {
        const bf16* src = WHAT == FWD ? a.x : a.dy;
        const long ld = WHAT == FWD ? a.ldx : a.ldy;
#pragma unroll
        for (int u = 0; u < UX; ++u) {
            int i = lo + u * 64 + r0;
            i = i < hi ? i : hi - 1;                       // rows behind the tile's last feed results nobody stores
            int row = a.rows ? a.rows[i] : i;
            row = (unsigned)row < (unsigned)a.T ? row : 0;
            px[u] = src + row * ld + cc;
        }
        const bf16* wbase = a.w + (long)(e < a.E ? e : 0) * a.stride_w;
#pragma unroll
        for (int u = 0; u < UY; ++u) {
            if constexpr (YK) py[u] = wbase + r0 * a.ldw + min(j0 + u * 64 + ck, NJ - 8);
            else py[u] = wbase + min(j0 + u * 64 + r0, NJ - 1) * a.ldw + cc;
        }
    } else {
#pragma unroll
        for (int u = 0; u < UX; ++u) px[u] = a.dy + min(i0 + u * 64 + ck, a.N - 8);
#pragma unroll
        for (int u = 0; u < UY; ++u) py[u] = a.x + min(j0 + u * 64 + ck, a.K - 8);
    }
    // what the results need, fetched before the loop: the output rows of a wave's stores and the bias of its columns
    constexpr int SEG = BN / 16;                           // sixteen-byte pieces of a wave's row
    constexpr int STORES = 16 * FH * SEG / 64;
    int orow[STORES];
    f32x4 bv[FN];
    if constexpr (WHAT != DW) {
#pragma unroll
        for (int q = 0; q < STORES; ++q) {
            const int i = lo + (wm * FM + kg * FH) * 16 + (q * 64 + lane) / SEG;
            orow[q] = i < hi ? (a.rows ? a.rows[i] : i) : -1;
        }
        const float* bias = WHAT == FWD && a.bias && e < a.E ? a.bias + (long)e * a.stride_b : nullptr;
#pragma unroll
        for (int n = 0; n < FN; ++n) {
            const int j = j0 + (wn * FN + n) * 16 + g * 4;
            bv[n] = bias && j < NJ ? *reinterpret_cast<const f32x4*>(bias + j) : f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    // in a vector register and opaque: a lane picks between two addresses, not between two loads
    const void* zeros = kZeros;
    asm volatile("" : "+v"(zeros));
    const bf16x8 ones = {(bf16)1.f, (bf16)1.f, (bf16)1.f, (bf16)1.f, (bf16)1.f, (bf16)1.f, (bf16)1.f, (bf16)1.f};

    const int chunk = XK && a.rows ? LIST / BK : kt1 - kt0 + 1;
    for (int c0 = kt0; c0 < kt1; c0 += chunk) {
        const int c1 = min(kt1, c0 + chunk), nk = c1 - c0;
        if constexpr (XK) {
            if (a.rows) {
                __syncthreads();                           // the last chunk's list has been read
                const int n = min(k_end - c0 * BK, LIST);
                for (int i = tid; i < n; i += THREADS) list[i] = a.rows[lo + c0 * BK + i];
                __syncthreads();
            }
        }
        auto stage = [&](int t, int st) {                  // K tile c0 + t
            char* dst = lds + st * STAGE + wave * 1024;
            if constexpr (WHAT == DW) {
                const int k0 = (c0 + t) * BK;
                const int k = k0 + r0;
                bool in = t < nk && k < k_end;
                long row = 0;
                if (in) {
                    const int r = a.rows ? list[t * BK + r0] : lo + k;
                    in = (unsigned)r < (unsigned)a.T;
                    row = r;
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const bf16* p = u < UX ? px[u] + row * a.ldy : py[u - UX] + row * a.ldx;
                    dma16(in ? (const void*)p : zeros, dst + u * UNIT);
                }
            } else {
                const int k0 = (c0 + t) * BK;
                const bool inx = k0 + cc < k_end && t < nk;
#pragma unroll
                for (int u = 0; u < UX; ++u) dma16(inx ? (const void*)(px[u] + k0) : zeros, dst + u * UNIT);
                const bool iny = YK ? k0 + r0 < k_end && t < nk : inx;
                const long step = YK ? k0 * a.ldw : k0;
#pragma unroll
                for (int u = 0; u < UY; ++u) dma16(iny ? (const void*)(py[u] + step) : zeros, dst + (UX + u) * UNIT);
            }
        };
#pragma unroll
        for (int t = 0; t < S; ++t) stage(t, t);
        // the fragments of K tile t + 1 come out of LDS while tile t is multiplied: two sets of registers
        struct Frags { bf16x8 x[FM], y[FN]; };
        auto fetch = [&](Frags& f, int st) {
            const char* lx = lds + st * STAGE;
#pragma unroll
            for (int m = 0; m < FM; ++m) f.x[m] = frag<XK>(lx, wm * FM + m, kg, lane);
#pragma unroll
            for (int n = 0; n < FN; ++n) f.y[n] = frag<YK>(lx + UX * UNIT, wn * FN + n, kg, lane);
        };
        auto fetched = [&](Frags& f) {
            lds_fence(f.x);
            lds_fence(f.y);
        };
        int cur = 0, nxt = 1;
        auto step = [&](int t, Frags& f, Frags& next) {
            // K tile t is in registers everywhere behind the barrier, so its stage takes the loads of K tile t + S
            wait_vm<(S - 2) * U>();                        // this wave's loads of K tile t + 1 have landed
            __builtin_amdgcn_s_barrier();                  // everybody's have
            asm volatile("" ::: "memory");
            fetch(next, nxt);
            stage(t + S, cur);
            __builtin_amdgcn_sched_barrier(0);             // reads and loads first: they run under the matrix instructions
#pragma unroll
            for (int m = 0; m < FM; ++m)
#pragma unroll
                for (int n = 0; n < FN; ++n)
                    acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.y[n], f.x[m], acc[m][n], 0, 0, 0);
            if constexpr (WHAT == DW) {
                if (sums) {
#pragma unroll
                    for (int m = 0; m < FM; ++m) rs[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, f.x[m], rs[m], 0, 0, 0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            fetched(next);
            cur = nxt;
            nxt = nxt == S - 1 ? 0 : nxt + 1;
        };
        Frags fa, fb;
        wait_vm<(S - 1) * U>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        fetch(fa, 0);
        fetched(fa);
#pragma unroll 1
        for (int t = 0; t + 1 < nk; t += 2) {
            step(t, fa, fb);
            step(t + 1, fb, fa);
        }
        if (nk & 1) step(nk - 1, fa, fb);
        wait_vm<0>();                                      // no load may land in LDS that is used for something else
        __syncthreads();
    }
    // the two halves of the reduction meet: group kg keeps the fragment rows kg FH .. kg FH + FH - 1 of its block
    {
        char* mine = lds + wave * (FH * FN * 1024) + lane * 16;
        const char* other = lds + (wave ^ 4) * (FH * FN * 1024) + lane * 16;
#pragma unroll
        for (int m = 0; m < FH; ++m)
#pragma unroll
            for (int n = 0; n < FN; ++n)
                *reinterpret_cast<f32x4*>(mine + (m * FN + n) * 1024) = kg ? acc[m][n] : acc[FH + m][n];
        if constexpr (XK) {
            if (sums && g == 0) {
#pragma unroll
                for (int m = 0; m < FM; ++m) sums_half[(wave * FM + m) * 16 + li] = rs[m][0];
            }
        }
        __syncthreads();
#pragma unroll
        for (int m = 0; m < FH; ++m)
#pragma unroll
            for (int n = 0; n < FN; ++n) {
                const f32x4 v = *reinterpret_cast<const f32x4*>(other + (m * FN + n) * 1024);
                acc[m][n] = (kg ? acc[FH + m][n] : acc[m][n]) + v;
            }
    }
    // a lane holds C[row li of fragment m][4 g .. 4 g + 3 of fragment n]
    if constexpr (WHAT == DW) {
        const long plane = (long)a.N * a.K;
        float* out = a.dw + ((long)slice * a.E + e) * plane;
#pragma unroll
        for (int m = 0; m < FH; ++m) {
            const int f = kg * FH + m, i = i0 + (wm * FM + f) * 16 + li;
#pragma unroll
            for (int n = 0; n < FN; ++n) {
                const int j = j0 + (wn * FN + n) * 16 + g * 4;
                if (i < a.N && j < a.K) *reinterpret_cast<f32x4*>(out + (long)i * a.K + j) = acc[m][n];
            }
            if (sums && g == 0 && i < a.N)
                a.db[((long)slice * a.E + e) * a.N + i] =
                    sums_half[(wave * FM + f) * 16 + li] + sums_half[((wave ^ 4) * FM + f) * 16 + li];
        }
    } else {
        __syncthreads();                                   // everybody has read the other half
        // through a patch of LDS of the wave's own, so that a lane stores sixteen bytes of a row
        char* patch = lds + wave * PATCH;
#pragma unroll
        for (int m = 0; m < FH; ++m)
#pragma unroll
            for (int n = 0; n < FN; ++n) {
                const f32x4 v = acc[m][n] + bv[n];
                *reinterpret_cast<bf16x4*>(patch + (m * 16 + li) * PITCH + n * 32 + g * 8) = pack4(v[0], v[1], v[2], v[3]);
            }
#pragma unroll
        for (int q = 0; q < STORES; ++q) {
            const int at = q * 64 + lane, r = at / SEG, c = at % SEG, j = j0 + wn * (BN / 2) + c * 8;
            const bf16x8 v = *reinterpret_cast<const bf16x8*>(patch + r * PITCH + c * 16);
            if ((unsigned)orow[q] < (unsigned)a.T && j < NJ)
                *reinterpret_cast<bf16x8*>((bf16*)a.out + orow[q] * a.ldo + j) = v;
        }
    }
}

// ------------------------------------------------------------------ dx over a short reduction
// dx = dy W with N a few K tiles: a 128 x 128 tile is over before its first loads have paid for themselves (5 us for 0.2 to
// 1 us of matrix instructions).  Here a workgroup keeps its rows of dy in LDS (BM rows, all of N) and runs through a
// chunk of columns of W without a stop: the loads of the next column tile are in flight while one is finished and stored.
// Stores that have no row or column go to a sink, so that their number, which the counted waits rely on, is known.
// Measured: 6144 rows, 320 -> 5120, six experts 36 us (63 MB written, 560 TFLOP/s).
__device__ float g_sink[256];
constexpr int DX_KX = 5;       // K tiles of dy that fit beside four stages of W

template <int BM, int KX>
__global__ __launch_bounds__(THREADS, 2) void grouped_dx_kernel(Args a, int tiles_j, int chunk_j) {
    constexpr int UX = BM / 64, WM = 2, WN = 4, FM = BM / WM / 16, FN = 128 / WN / 16, RS = 4, UY = 2;
    constexpr int SEG = FN * 2, STORES = FM * 16 * SEG / 64, PITCH = FN * 32 + 16, PATCH = 16 * PITCH;
    // ONE array: with three, the compiler tells their reads from the loads into them apart and waits for all of them before
    // the first read of a step
    __shared__ __attribute__((aligned(16))) char lds[(KX * UX + RS * UY) * UNIT + 8 * PATCH];
    char* const xs = lds;
    char* const ys = lds + KX * UX * UNIT;
    char* const patches = ys + RS * UY * UNIT;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN, g = lane >> 4, li = lane & 15;
    const int chunks = (tiles_j + chunk_j - 1) / chunk_j;
    int lo, hi, jt0;
    const int e = find_tile(a, BM, chunks, lane, lo, hi, jt0);
    if (e < 0) return;
    jt0 *= chunk_j;
    const int nj = min(chunk_j, tiles_j - jt0);
    const int kx = e == a.E ? 0 : (a.N + BK - 1) / BK;
    bf16* optr[STORES];                                    // where a lane's pieces go, but for the column
    bool ok[STORES];
#pragma unroll
    for (int q = 0; q < STORES; ++q) {
        const int i = lo + wm * FM * 16 + (q * 64 + lane) / SEG;
        const int row = i < hi ? (a.rows ? a.rows[i] : i) : -1;
        ok[q] = (unsigned)row < (unsigned)a.T;
        optr[q] = (bf16*)a.out + (ok[q] ? row : 0) * a.ldo + (jt0 * 128 + wn * FN * 16 + (q * 64 + lane) % SEG * 8);
    }
    const int jcol = jt0 * 128 + wn * FN * 16 + lane % SEG * 8;    // (64 is a multiple of SEG)
    uintptr_t sink = (uintptr_t)(g_sink + lane * 4);
    const void* zeros = kZeros;
    asm volatile("" : "+v"(zeros), "+v"(sink));
    auto store = [&](int jt, int q, bf16x8 v) {
        store_at(ok[q] && jcol + jt * 128 < a.K ? (uintptr_t)(optr[q] + jt * 128) : sink, v);
    };
    if (kx == 0) {                                         // rows that no expert takes
        for (int jt = 0; jt < nj; ++jt)
#pragma unroll
            for (int q = 0; q < STORES; ++q) store(jt, q, bf16x8{});
        return;
    }
    const int r0 = tid >> 3;
    const int cc = ((tid & 7) ^ (r0 & 7)) * 8;
    const int ck = ((((tid & 7) >> 1) ^ kmaj_key(r0)) * 2 + (tid & 1)) * 8;
    {
        const bf16* px[UX];
#pragma unroll
        for (int u = 0; u < UX; ++u) {
            const int i = min(lo + u * 64 + r0, hi - 1);
            int row = a.rows ? a.rows[i] : i;
            row = (unsigned)row < (unsigned)a.T ? row : 0;
            px[u] = a.dy + row * a.ldy + cc;
        }
        for (int kt = 0; kt < kx; ++kt)
#pragma unroll
            for (int u = 0; u < UX; ++u)
                dma16(kt * BK + cc < a.N ? (const void*)(px[u] + kt * BK) : zeros, xs + (kt * UX + u) * UNIT + wave * 1024);
    }
    const bf16* wrow = a.w + (long)e * a.stride_w + r0 * a.ldw;
    const int steps = nj * kx;
    int sj = 0, sk = 0;                                    // column tile and K tile of the next load
    auto stage = [&](int st) {
        const bool in = sj < nj && sk * BK + r0 < a.N;
        const bf16* p = wrow + sk * BK * a.ldw;
#pragma unroll
        for (int u = 0; u < UY; ++u) {
            const int col = min((jt0 + sj) * 128 + u * 64 + ck, a.K - 8);
            dma16(in ? (const void*)(p + col) : zeros, ys + (st * UY + u) * UNIT + wave * 1024);
        }
        if (++sk == kx) { sk = 0; ++sj; }
    };
    f32x4 acc[FM][FN];
#pragma unroll
    for (int m = 0; m < FM; ++m)
#pragma unroll
        for (int n = 0; n < FN; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    struct Frags { bf16x8 x[FM][2], y[FN][2]; };
    auto fetch = [&](Frags& f, int kt, int st) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int m = 0; m < FM; ++m) f.x[m][s] = frag<false>(xs + kt * UX * UNIT, wm * FM + m, s, lane);
#pragma unroll
            for (int n = 0; n < FN; ++n) f.y[n][s] = frag<true>(ys + st * UY * UNIT, wn * FN + n, s, lane);
        }
    };
    int fk = 0, fs = 0;                                    // K tile and ring slot of the next fragments
    int cj = 0, ck_ = 0, cs = 0;                           // column tile, K tile and ring slot being multiplied
    auto advance = [&]() {
        if (++fk == kx) fk = 0;
        if (++fs == RS) fs = 0;
    };
    auto step = [&](Frags& f, Frags& next, auto stored) {
        // K tile + 1 of W has landed: behind it are the loads of one more and, right after a column tile, its stores
        if constexpr (decltype(stored)::value) wait_vm<(RS - 2) * UY + STORES>();
        else wait_vm<(RS - 2) * UY>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        fetch(next, fk, fs);
        advance();
        stage(cs);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int m = 0; m < FM; ++m)
#pragma unroll
                for (int n = 0; n < FN; ++n)
                    acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.y[n][s], f.x[m][s], acc[m][n], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        lds_fence(next.x);
        lds_fence(next.y);
        if (++cs == RS) cs = 0;
    };
    auto finish = [&]() {                                  // one column tile: through a patch of the wave's own to sixteen bytes a lane
        char* patch = patches + wave * PATCH;
#pragma unroll
        for (int m = 0; m < FM; ++m) {
#pragma unroll
            for (int n = 0; n < FN; ++n) {
                *reinterpret_cast<bf16x4*>(patch + li * PITCH + n * 32 + g * 8) =
                    pack4(acc[m][n][0], acc[m][n][1], acc[m][n][2], acc[m][n][3]);
                acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
#pragma unroll
            for (int q = 0; q < STORES / FM; ++q) {
                const int at = q * 64 + lane;
                store(cj, m * (STORES / FM) + q, *reinterpret_cast<const bf16x8*>(patch + at / SEG * PITCH + at % SEG * 16));
            }
        }
        ++cj;
    };
    for (int s = 0; s < RS; ++s) stage(s);
    Frags fa, fb;
    wait_vm<(RS - 1) * UY>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    fetch(fa, fk, fs);
    advance();
    lds_fence(fa.x);
    lds_fence(fa.y);
    bool stored = false;
#pragma unroll 1
    for (int s = 0; s < steps; s += 2) {
        if (stored) step(fa, fb, std::true_type{});
        else step(fa, fb, std::false_type{});
        stored = ++ck_ == kx;
        if (stored) { ck_ = 0; finish(); }
        if (s + 1 >= steps) break;
        if (stored) step(fb, fa, std::true_type{});
        else step(fb, fa, std::false_type{});
        stored = ++ck_ == kx;
        if (stored) { ck_ = 0; finish(); }
    }
    wait_vm<0>();                                          // no load may outlive the workgroup
}

// ------------------------------------------------------------------ few rows
// Forward product of few rows: what counts is how soon the weights have been read, by how many CUs.  A workgroup computes
// 16 FM rows x 16 FN columns; its eight waves take every eighth chunk of 64 reduction steps straight from memory into
// matrix-instruction operands (nobody else in the workgroup reads the same bytes, so LDS would only add a stop), four
// chunks in flight each, and the eight partial tiles are added up in LDS in a fixed order.  Measured: one row of K 1536, N 96 5.4 us,
// of which a launch that does nothing takes about 2; 192 rows of K 4096, N 256 12 us.
template <int FM, int FN>
__global__ __launch_bounds__(THREADS, 2) void grouped_narrow_kernel(Args a, int tiles_j) {
    constexpr int TM = 16 * FM, TN = 16 * FN, DEEP = FM + FN > 4 ? 2 : 4;
    __shared__ __attribute__((aligned(16))) float part[8][TM][TN + 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, li = lane & 15;
    int lo, hi, j0;
    const int e = find_tile(a, TM, tiles_j, lane, lo, hi, j0);
    if (e < 0) return;
    j0 *= TN;
    f32x4 acc[FM][FN];
#pragma unroll
    for (int m = 0; m < FM; ++m)
#pragma unroll
        for (int n = 0; n < FN; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (e < a.E) {
        const bf16 *px[FM], *py[FN];
#pragma unroll
        for (int m = 0; m < FM; ++m) {
            const int i = min(lo + m * 16 + li, hi - 1);
            int row = a.rows ? a.rows[i] : i;
            row = (unsigned)row < (unsigned)a.T ? row : 0;
            px[m] = a.x + row * a.ldx + g * 8;
        }
#pragma unroll
        for (int n = 0; n < FN; ++n)
            py[n] = a.w + (long)e * a.stride_w + min(j0 + n * 16 + li, a.N - 1) * a.ldw + g * 8;
        uintptr_t zeros = (uintptr_t)kZeros;
        asm volatile("" : "+v"(zeros));
        const int chunks = (a.K + 63) / 64;
        for (int c0 = wave; c0 < chunks; c0 += 8 * DEEP) {
            bf16x8 xf[DEEP][FM][2], yf[DEEP][FN][2];
#pragma unroll
            for (int d = 0; d < DEEP; ++d)
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const int k = (c0 + 8 * d) * 64 + s * 32;
                    const bool in = k + g * 8 < a.K;
#pragma unroll
                    for (int m = 0; m < FM; ++m)
                        xf[d][m][s] = load_at<bf16x8>(in ? (uintptr_t)(px[m] + k) : zeros);
#pragma unroll
                    for (int n = 0; n < FN; ++n)
                        yf[d][n][s] = load_at<bf16x8>(in ? (uintptr_t)(py[n] + k) : zeros);
                }
            __builtin_amdgcn_sched_barrier(0);             // all loads of a round are on their way before the first is used
#pragma unroll
            for (int d = 0; d < DEEP; ++d)
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int m = 0; m < FM; ++m)
#pragma unroll
                        for (int n = 0; n < FN; ++n)
                            acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(yf[d][n][s], xf[d][m][s], acc[m][n], 0, 0, 0);
        }
    }
#pragma unroll
    for (int m = 0; m < FM; ++m)
#pragma unroll
        for (int n = 0; n < FN; ++n) *reinterpret_cast<f32x4*>(&part[wave][m * 16 + li][n * 16 + g * 4]) = acc[m][n];
    __syncthreads();
    for (int q = tid; q < TM * TN / 4; q += THREADS) {
        const int r = q / (TN / 4), c = q % (TN / 4) * 4, i = lo + r, j = j0 + c;
        if (i >= hi || j >= a.N) continue;
        const int row = a.rows ? a.rows[i] : i;
        if ((unsigned)row >= (unsigned)a.T) continue;
        f32x4 v = *reinterpret_cast<const f32x4*>(&part[0][r][c]);
#pragma unroll
        for (int w = 1; w < 8; ++w) v += *reinterpret_cast<const f32x4*>(&part[w][r][c]);
        if (a.bias && e < a.E) v += *reinterpret_cast<const f32x4*>(a.bias + (long)e * a.stride_b + j);
        *reinterpret_cast<bf16x4*>((bf16*)a.out + row * a.ldo + j) = pack4(v[0], v[1], v[2], v[3]);
    }
}

// dw[i], then db[i] = sum over the slices, in order (float4s; part holds the slices of dW, then those of db)
__global__ __launch_bounds__(256) void slice_sum_kernel(const f32x4* __restrict__ part, f32x4* __restrict__ dw, long n,
                                                        f32x4* __restrict__ db, long nb, int slices) {
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n + nb; i += (long)gridDim.x * 256) {
        const bool bias = i >= n;
        const f32x4* p = bias ? part + slices * n + (i - n) : part + i;
        const long step = bias ? nb : n;
        f32x4 v = p[0];
        for (int s = 1; s < slices; ++s) v += p[s * step];
        if (bias) db[i - n] = v;
        else dw[i] = v;
    }
}

// ------------------------------------------------------------------ rows in the order of their experts
constexpr int SORT_THREADS = 1024, SORT_WAVES = 16, SORT_MAX_E = 512, SORT_DEEP = 16;

// lanes of the wave with this lane's key (keys below 2^bits)
__device__ __forceinline__ unsigned long long same_key(int key, int bits) {
    unsigned long long mask = ~0ull;
    for (int b = 0; b < bits; ++b) {
        const unsigned long long one = __ballot((key >> b) & 1);
        mask &= ((key >> b) & 1) ? one : ~one;
    }
    return mask;
}

// Stable counting sort by one workgroup: every wave walks a run of consecutive rows twice, first counting per key, then --
// after a scan over (key, wave) -- writing.  Keys are experts, E for a row that none takes.  The time is that of the loads,
// one after the other 1 us each, so sixteen times 64 rows are fetched at once; up to 16384 rows a wave then has all of its
// keys in registers for both walks.
__global__ __launch_bounds__(SORT_THREADS) void expert_rows_kernel(const int* __restrict__ expert, int T, int E, int bits,
                                                                   int* __restrict__ rows, int* __restrict__ offsets) {
    __shared__ int count[SORT_WAVES][SORT_MAX_E + 1];
    __shared__ int wave_total[SORT_WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, keys = E + 1;
    const int chunks = (T + 63) / 64, each = (chunks + SORT_WAVES - 1) / SORT_WAVES;
    const int c0 = wave * each, c1 = min(c0 + each, chunks);
    int key[SORT_DEEP];
    auto fetch = [&](int c) {
#pragma unroll
        for (int d = 0; d < SORT_DEEP; ++d) {
            const int t = (c + d) * 64 + lane;
            key[d] = -1;                               // no row
            if (c + d < c1 && t < T) key[d] = expert[t];
            else continue;
            key[d] = (unsigned)key[d] < (unsigned)E ? key[d] : E;
        }
    };
    fetch(c0);
    for (int i = lane; i < keys; i += 64) count[wave][i] = 0;
    for (int c = c0; c < c1; c += SORT_DEEP) {
        if (c > c0) fetch(c);
#pragma unroll
        for (int d = 0; d < SORT_DEEP; ++d) {
            if (c + d >= c1) break;
            const bool in = key[d] >= 0;
            const unsigned long long mask = same_key(key[d], bits) & __ballot(in);
            if (in && lane == __builtin_ctzll(mask)) count[wave][key[d]] += __popcll(mask);
        }
    }
    __syncthreads();
    // exclusive scan in the order (key, wave): thread k owns key k
    int mine = 0;
    if (tid < keys)
#pragma unroll
        for (int w = 0; w < SORT_WAVES; ++w) mine += count[w][tid];
    const int sum = wave_scan(mine);
    if (lane == 63) wave_total[wave] = sum;
    __syncthreads();
    int base = sum - mine;
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) base += w < wave ? wave_total[w] : 0;
    if (tid < keys) {
        offsets[tid] = base;                       // key E: the end of the last expert's rows
#pragma unroll
        for (int w = 0; w < SORT_WAVES; ++w) {
            const int n = count[w][tid];
            count[w][tid] = base;
            base += n;
        }
    }
    __syncthreads();
    for (int c = c0; c < c1; c += SORT_DEEP) {
        if (each > SORT_DEEP) fetch(c);
#pragma unroll
        for (int d = 0; d < SORT_DEEP; ++d) {
            if (c + d >= c1) break;
            const bool in = key[d] >= 0;
            const unsigned long long mask = same_key(key[d], bits) & __ballot(in);
            if (in) {
                const int at = count[wave][key[d]];    // every lane of the key reads before its first lane moves it on
                rows[at + __popcll(mask & ((1ull << lane) - 1))] = (c + d) * 64 + lane;
                if (lane == __builtin_ctzll(mask)) count[wave][key[d]] = at + __popcll(mask);
            }
        }
    }
}

// The same for fewer than FEW_KEYS experts and many rows: a lane owns a run of consecutive rows and a counter per key (in LDS, its
// own column: no conflicts), so that a row costs a lane a few instructions instead of costing a wave a round of votes; the
// scans over the lanes, one per key, are what it costs beyond that.  us at 192 / 5003 / 12288 rows, votes against runs: 6 experts 3.4 /
// 7.1 / 13, 4.9 / 5.5 / 6.2; 24 experts 3.5 / 8.3 / 15.8, 6.9 / 7.9 / 10.0.
// The list itself is put together in LDS where it fits beside the counters (KEYS of 16, up to 16384 rows), so that what leaves are
// whole lines.
constexpr int FEW_KEYS = 32, FEW_ROWS = 16384;

template <int KEYS>
__global__ __launch_bounds__(SORT_THREADS) void expert_rows_few_kernel(const int* __restrict__ expert, int T, int E,
                                                                       int* __restrict__ rows, int* __restrict__ offsets) {
    constexpr int LIST = KEYS <= 16 ? FEW_ROWS : 1;
    __shared__ int count[KEYS][SORT_THREADS];
    __shared__ int total[SORT_WAVES][KEYS];
    __shared__ int list[LIST];
    const bool staged = T <= LIST;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, keys = E + 1;
    const int each = ((T + SORT_THREADS - 1) / SORT_THREADS + 3) & ~3;      // whole sixteen-byte loads
    const int t0 = min((long)tid * each, (long)T), t1 = min(t0 + each, T);
    const bool wide = ((uintptr_t)expert & 15) == 0;
    int key[SORT_DEEP];
    auto fetch = [&](int t) {
#pragma unroll
        for (int d = 0; d < SORT_DEEP; d += 4) {
            int4 v = make_int4(E, E, E, E);
            if (wide && t + d + 3 < t1) {
                v = *reinterpret_cast<const int4*>(expert + t + d);
            } else {
                if (t + d < t1) v.x = expert[t + d];
                if (t + d + 1 < t1) v.y = expert[t + d + 1];
                if (t + d + 2 < t1) v.z = expert[t + d + 2];
                if (t + d + 3 < t1) v.w = expert[t + d + 3];
            }
            key[d] = v.x; key[d + 1] = v.y; key[d + 2] = v.z; key[d + 3] = v.w;
        }
#pragma unroll
        for (int d = 0; d < SORT_DEEP; ++d) key[d] = (unsigned)key[d] < (unsigned)E ? key[d] : E;
    };
    fetch(t0);
    for (int k = 0; k < keys; ++k) count[k][tid] = 0;
    for (int t = t0; t < t0 + each; t += SORT_DEEP) {
        if (each > SORT_DEEP) fetch(t);
#pragma unroll
        for (int d = 0; d < SORT_DEEP; ++d)
            if (t + d < t1) __hip_atomic_fetch_add(&count[key[d]][tid], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
    // (a lane's counters are its own, and LDS works a wave's instructions off in order: no barrier before it reads them
    // back; the additions carry no order between lanes, they are additions because those need no round trip)
#pragma unroll 4
    for (int k = 0; k < keys; ++k) {
        const int n = count[k][tid], sum = wave_scan(n);
        count[k][tid] = sum - n;
        if (lane == 63) total[wave][k] = sum;
    }
    __syncthreads();
    if (tid < 64) {                                    // where the rows of (key, wave) begin: lane k owns key k
        int n[SORT_WAVES], mine = 0;
#pragma unroll
        for (int w = 0; w < SORT_WAVES; ++w) {
            n[w] = lane < keys ? total[w][lane] : 0;
            mine += n[w];
        }
        int base = wave_scan(mine) - mine;
        if (lane < keys) {
            offsets[lane] = base;                      // key E: the end of the last expert's rows
#pragma unroll
            for (int w = 0; w < SORT_WAVES; ++w) {
                total[w][lane] = base;
                base += n[w];
            }
        }
    }
    __syncthreads();
    for (int t = t0; t < t0 + each; t += SORT_DEEP) {
        if (each > SORT_DEEP) fetch(t);
#pragma unroll
        for (int d = 0; d < SORT_DEEP; ++d)
            if (t + d < t1) {
                const int at = __hip_atomic_fetch_add(&count[key[d]][tid], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                const int to = total[wave][key[d]] + at;
                if (staged) list[to] = t + d;
                else rows[to] = t + d;
            }
    }
    if (!staged) return;
    __syncthreads();
    for (int i = tid; i < T; i += SORT_THREADS) rows[i] = list[i];
}

constexpr int MAX_T = 1 << 30;                         // row and column numbers, and a tile or a run behind them, stay in 32 bits

int cdiv(long a, long b) { return (int)((a + b - 1) / b); }

}  // namespace

extern "C" int vp_expert_rows(const int* expert, int T, int E, int* rows, int* offsets, hipStream_t stream) {
    VP_CHECK_ARG(T >= 0 && T <= MAX_T && E >= 1 && offsets && (T == 0 || (expert && rows)));
    if (E > SORT_MAX_E) return VP_ERR_UNSUPPORTED;
    if (E < FEW_KEYS && T > 1800 + 110 * E) {       // (where the two measured the same)
        auto kernel = E < 16 ? expert_rows_few_kernel<16> : expert_rows_few_kernel<FEW_KEYS>;
        hipLaunchKernelGGL(kernel, dim3(1), dim3(SORT_THREADS), 0, stream, expert, T, E, rows, offsets);
        VP_LAUNCH_RET();
    }
    int bits = 1;
    while ((1 << bits) <= E) ++bits;
    hipLaunchKernelGGL(expert_rows_kernel, dim3(1), dim3(SORT_THREADS), 0, stream, expert, T, E, bits, rows, offsets);
    VP_LAUNCH_RET();
}

namespace {

int check_common(const vp_grouped_args* g) {
    VP_CHECK_ARG(g && g->T >= 0 && g->T <= MAX_T && g->E >= 1 && g->N >= 8 && g->K >= 8 && g->N % 8 == 0 && g->K % 8 == 0 && g->offsets);
    VP_CHECK_ARG(g->N <= MAX_T && g->K <= MAX_T);
    return VP_OK;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

Args make_args(const vp_grouped_args* g) {
    Args a{};
    a.offsets = g->offsets; a.rows = g->rows;
    a.T = g->T; a.E = g->E; a.N = g->N; a.K = g->K;
    a.x = (const bf16*)g->x; a.ldx = g->ldx;
    a.w = (const bf16*)g->w; a.ldw = g->ldw; a.stride_w = g->stride_w;
    a.bias = g->bias; a.stride_b = g->stride_b;
    a.dy = (const bf16*)g->dy; a.ldy = g->ldy;
    a.out = g->out; a.ldo = g->ldo;
    a.zero_rest = g->zero_rest;
    a.slices = 1;
    return a;
}

// upper bound of the row tiles: every expert's last tile may be partial; rows behind the last expert and before the first add
// one more each
int row_tiles(const vp_grouped_args* g, int bm) {
    const long groups = (long)g->E < g->T ? g->E : g->T;
    return (int)(g->T / bm + groups + (g->zero_rest ? 2 : 0));
}

// Row tiles that there will probably be: experts' last tiles are half full on average, of many experts' a little less, and every
// expert with a row has one.
long likely_tiles(const vp_grouped_args* g, int bm) {
    const long e = std::min(g->E, g->T);
    return std::max(g->T / bm + (e + 1) / 2 + e / 8, e);
}

// Operand rows that n tiles of 64 x 128 cost a CU, two of which share one: a round of 512, the first 256, more of the last round
long shared_cost(long n, long round, long most) {
    return n / 512 * round + (n % 512 == 0 ? 0 : n % 512 <= 256 ? 200 : most);
}

template <int FM, int FN>
int launch_narrow(const vp_grouped_args* g, hipStream_t stream) {
    const int tj = cdiv(g->N, 16 * FN);
    const long grid = (long)row_tiles(g, 16 * FM) * tj;
    if (!grid_fits(grid, THREADS)) return VP_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((grouped_narrow_kernel<FM, FN>), dim3((unsigned)grid), dim3(THREADS), 0, stream, make_args(g), tj);
    VP_LAUNCH_RET();
}

// Workgroups a row tile: as many column chunks as finish first, a workgroup costing its column tiles (kx K tiles and about
// two more for the stores) and about six K tiles to begin.
int launch_dx(const vp_grouped_args* g, hipStream_t stream) {
    constexpr int BM = 128, KX = DX_KX;
    const int tj = cdiv(g->K, 128), kx = cdiv(g->N, BK);
    const long tiles = likely_tiles(g, BM);
    int chunk = tj;
    long best = -1;
    for (int c = 1; c <= tj; ++c) {
        const int each = cdiv(tj, c);
        if (!grid_fits((long)row_tiles(g, BM) * cdiv(tj, each), THREADS)) continue;
        const long cost = (tiles * cdiv(tj, each) + 255) / 256 * (each * (kx + 2) + 6);
        if (best < 0 || cost < best) { best = cost; chunk = each; }
    }
    const long grid = (long)row_tiles(g, BM) * cdiv(tj, chunk);
    if (!grid_fits(grid, THREADS)) return VP_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((grouped_dx_kernel<BM, KX>), dim3((unsigned)grid), dim3(THREADS), 0, stream, make_args(g), tj, chunk);
    VP_LAUNCH_RET();
}

template <int WHAT, int BM, int S, int PER_CU = 1, int BN = 128>
int launch_rows(const vp_grouped_args* g, hipStream_t stream) {
    const int tj = cdiv(WHAT == FWD ? g->N : g->K, BN);
    const long grid = (long)row_tiles(g, BM) * tj;
    if (!grid_fits(grid, THREADS)) return VP_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((grouped_kernel<WHAT, BM, BN, S, PER_CU>), dim3((unsigned)grid), dim3(THREADS), 0, stream, make_args(g), tj, 0);
    VP_LAUNCH_RET();
}

// dW in tiles of 64 x 128, two of which share a CU: one's loads and stores pass under the other's sums, and an extent of N that
// ends in the first half of 128 wastes nothing.  us at 32 / 768 / 5003 / 12288 rows against one 128 x 128 (N 320: 64 x 256) tile a CU:
// 5120 x 320, six experts 19 / 21 / 40 / 91 against 22 / 25 / 40 / 93; 4096 x 256 13 / 16 / 28 / 63, 15 / 17 / 29 / 64; 1024 x 1024, 24
// experts 33 / 42 / 54 / 76, 35 / 45 / 60 / 76; 512 x 512, 48 experts 22 / 28 / 32 / 37, 22 / 28 / 35 / 39.
constexpr int DW_BM = 64, DW_BN = 128;

// The rows are cut into slices where the tiles alone would leave CUs without work and the time that it saves, 6 us a thousand rows of
// the largest expert (say twice the mean), is more than the partial sums cost: 3.5 us of a launch and their way to memory and back.
// us in one slice / in what this chooses, skewed shares: 2500 rows of 224 x 1416, five experts 14 (19 in two), 96 x 3024, one expert
// 22 / 15, 4000 rows of 32 x 560, five experts 16 / 11.
int dw_slices(int T, int E, int N, int K) {
    const double rows = std::min((double)T, 2.0 * T / E), bytes = 4.0 * E * N * K;
    const long cap = std::min<long>(512 / std::max<long>((long)E * cdiv(N, DW_BM) * cdiv(K, DW_BN), 1), (long)(rows / 256));
    int best = 1;
    double least = 6e-3 * rows;
    for (int s = 2; s <= cap; ++s) {
        const double us = 6e-3 * rows / s + 3.5 + 2 * s * bytes / 4.5e6;
        if (us < least) { least = us; best = s; }
    }
    return best;
}

}  // namespace

extern "C" int vp_grouped_fwd(const vp_grouped_args* g, hipStream_t stream) {
    if (int rc = check_common(g)) return rc;
    if (g->T == 0) return VP_OK;
    VP_CHECK_ARG(g->x && g->w && g->out && aligned16(g->x) && aligned16(g->w) && aligned16(g->out));
    VP_CHECK_ARG(g->ldx >= g->K && g->ldw >= g->K && g->ldo >= g->N && g->ldx % 8 == 0 && g->ldw % 8 == 0 && g->ldo % 8 == 0);
    VP_CHECK_ARG(g->stride_w % 8 == 0 && (!g->bias || (aligned16(g->bias) && g->stride_b % 4 == 0)));
    // The kernels differ in how many bytes a CU has to fetch: a workgroup reads tile rows + tile columns operand rows, 256 run
    // at a time, and a CU takes in some 50 KB a microsecond, whoever else is running -- twice that where the loads go to LDS
    // several K tiles ahead, as in the 128-wide tiles.  The smallest (rounds x operand rows) wins; it ranks what was measured
    // right.  K 4096, N 256, 6 experts, us at 1 / 192 / 768 / 1536 rows: 16 x 16 7.1 / 17.9 / 31.5 / 52, 16 x 32 10.9 / 15.0 / 25 / 46,
    // 32 x 32 12.2 / 18.6 / 18.9 / 34, 32 x 64 19.0 / 25.4 / 25.4 / 25.8, 128 x 128 31.1 / 32.0 / 32.4 / 32.5.  K 1024, N 1024, 24
    // experts at 1 / 96 / 768 rows: 4.3 / 20 / 49, 5.6 / 17.8 / 41, 6.4 / 22.5 / 44, 7.4 / 15.5 / 33, 11.6 / 14.1 / 15.3.
    // Of the 64 x 128 and the 128 x 64 tiles two share a CU: 200 rows up to 256 of them, then what the next lines say, measured with
    // inputs in memory.  us, 64 x 128 / 128 x 64 / 128 x 128 / 192 x 128 (three stages): K 5120, N 320 at 5003 rows 41 / 42 / 51 / 62, 6144
    // 64 / 44 / 53 / 63, 12288 96 / 79 / 95 / 67, 16384 117 / 110 / 101 / 119; K 4096, N 256 at 5003 34 / 34 / 41 / 51, 12288 59 / 60 / 47 / 55,
    // 16384 79 / 77 / 79 / 61; K 2048, N 1024, 8 experts at 12288 89 / - / 87 / 83, 16384 113 / - / 112 / 90.
    constexpr long NEVER = 1l << 62;                       // (more workgroups than a launch takes)
    const auto tiles = [&](int tm, int tn) { return likely_tiles(g, tm) * cdiv(g->N, tn); };
    const auto never = [&](int tm, int tn) { return grid_fits((long)row_tiles(g, tm) * cdiv(g->N, tn), THREADS) ? 0 : NEVER; };
    const auto cost = [&](int tm, int tn, int weight) { return (tiles(tm, tn) + 255) / 256 * (tm + tn) * weight + never(tm, tn); };
    const long c11 = cost(16, 16, 2), c12 = cost(16, 32, 2), c22 = cost(32, 32, 2), c24 = cost(32, 64, 2), c128 = cost(128, 128, 1);
    const long c192 = cost(192, 128, 1);
    const long c64 = shared_cost(tiles(64, 128), 285, 330) + never(64, 128), c64n = shared_cost(tiles(128, 64), 340, 390) + 1 + never(128, 64);
    const long best = std::min({c11, c12, c22, c24, c64, c64n, c128, c192});
    if (best >= NEVER) return VP_ERR_UNSUPPORTED;
    if (best == c11) return launch_narrow<1, 1>(g, stream);
    if (best == c12) return launch_narrow<1, 2>(g, stream);
    if (best == c22) return launch_narrow<2, 2>(g, stream);
    if (best == c24) return launch_narrow<2, 4>(g, stream);
    if (best == c64) return launch_rows<FWD, 64, 3, 2>(g, stream);
    if (best == c64n) return launch_rows<FWD, 128, 3, 2, 64>(g, stream);
    return best == c128 ? launch_rows<FWD, 128, 4>(g, stream) : launch_rows<FWD, 192, 3>(g, stream);
}

extern "C" int vp_grouped_dgrad(const vp_grouped_args* g, hipStream_t stream) {
    if (int rc = check_common(g)) return rc;
    if (g->T == 0) return VP_OK;
    VP_CHECK_ARG(g->dy && g->w && g->out && aligned16(g->dy) && aligned16(g->w) && aligned16(g->out));
    VP_CHECK_ARG(g->ldy >= g->N && g->ldw >= g->K && g->ldo >= g->K && g->ldy % 8 == 0 && g->ldw % 8 == 0 && g->ldo % 8 == 0);
    VP_CHECK_ARG(g->stride_w % 8 == 0);
    // us at 192 / 1536 / 6144 / 12288 rows (skewed shares) for W of 320 x 4096, six experts: columns in a run 9.6 / 16 / 31 / 62,
    // 64 x 128 tiles 7.8 / 17 / 44 / 81, 128 x 128 tiles 9.5 / 24 / 50 / 87.  Tiles as for the forward product, but for the shortest
    // reductions, where a tile is mostly beginning and end and small ones win: N 384 at 12288 rows 64 x 128 28, 192 x 128 31.  N 768,
    // K 4096, six experts at 1536 / 5003 / 12288 rows: 64 x 128 32 / 76 / 176, chosen 29 / 64 / 145; one expert, N 752, K 3384 at 5003 64 / 49.
    if (g->N <= DX_KX * BK) {
        const int rc = launch_dx(g, stream);
        if (rc != VP_ERR_UNSUPPORTED) return rc;
    }
    constexpr long NEVER = 1l << 62;
    const auto tiles = [&](int tm) { return likely_tiles(g, tm) * cdiv(g->K, 128); };
    const auto never = [&](int tm) { return grid_fits((long)row_tiles(g, tm) * cdiv(g->K, 128), THREADS) ? 0 : NEVER; };
    const long c64 = (g->N <= 384 ? 0 : shared_cost(tiles(64), 285, 330)) + never(64);
    const long c128 = (tiles(128) + 255) / 256 * 256 + never(128), c192 = (tiles(192) + 255) / 256 * 320 + never(192);
    if (std::min({c64, c128, c192}) >= NEVER) return VP_ERR_UNSUPPORTED;
    if (c64 <= std::min(c128, c192)) return launch_rows<DX, 64, 3>(g, stream);
    return c128 <= c192 ? launch_rows<DX, 128, 4>(g, stream) : launch_rows<DX, 192, 3>(g, stream);
}

extern "C" int vp_grouped_wgrad_slices(int T, int E, int N, int K) {
    return T < 0 || E < 1 || N < 8 || K < 8 ? 1 : dw_slices(T, E, N, K);
}

extern "C" int vp_grouped_wgrad(const vp_grouped_args* g, float* dw, float* db, void* workspace, size_t workspace_bytes,
                                hipStream_t stream) {
    if (int rc = check_common(g)) return rc;
    VP_CHECK_ARG(dw && aligned16(dw) && (g->T == 0 || (g->dy && g->x && aligned16(g->dy) && aligned16(g->x))));
    VP_CHECK_ARG(g->ldx >= g->K && g->ldy >= g->N && g->ldx % 8 == 0 && g->ldy % 8 == 0 && (!db || aligned16(db)));
    Args a = make_args(g);
    const int ti = cdiv(g->N, DW_BM), tj = cdiv(g->K, DW_BN);
    a.slices = dw_slices(g->T, g->E, g->N, g->K);
    const size_t need = a.slices == 1 ? 0 : (size_t)a.slices * g->E * g->N * ((size_t)g->K + (db ? 1 : 0)) * 4;
    VP_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && aligned16(workspace)));
    const long n = (long)g->E * g->N * g->K, nb = (long)g->E * g->N;
    a.dw = a.slices == 1 ? dw : (float*)workspace;
    a.db = a.slices == 1 ? db : (db ? (float*)workspace + a.slices * n : nullptr);
    const long grid = ((long)g->E * tj * a.slices + 7) / 8 * 8 * ti;
    if (!grid_fits(grid, THREADS)) return VP_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((grouped_kernel<DW, DW_BM, DW_BN, 3, 2>), dim3((unsigned)grid), dim3(THREADS), 0, stream, a, tj, ti);
    if (a.slices > 1) {
        const long n4 = n / 4, nb4 = db ? nb / 4 : 0;
        const int blocks = (int)std::min<long>((n4 + nb4 + 255) / 256, 2048);
        hipLaunchKernelGGL(slice_sum_kernel, dim3(blocks), dim3(256), 0, stream, (const f32x4*)workspace, (f32x4*)dw, n4, (f32x4*)db, nb4,
                           a.slices);
    }
    VP_LAUNCH_RET();
}
