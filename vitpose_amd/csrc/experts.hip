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
#include <type_traits>

#include "common.h"
#include "vitpose_hip.h"

namespace {

constexpr int BK = 64, UNIT = 64 * BK * 2, THREADS = 256;   // a unit: 64 rows (or columns) x 64 reduction steps, 8 KiB

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

// rows of expert e in the list, kept inside it whatever the offsets say
__device__ __forceinline__ Span span_of(const int* offsets, int e, int T) {
    int lo = offsets[e], hi = offsets[e + 1];
    lo = lo < 0 ? 0 : (lo > T ? T : lo);
    hi = hi < lo ? lo : (hi > T ? T : hi);
    return Span{lo, hi};
}

// Which expert's rows tile number `tile` of a launch holds: every wave scans the experts' tile counts, 64 at a time.
// Returns the expert (E: the rows behind the last expert, -1: none) and its first and last list entry.
__device__ __forceinline__ int find_tile(const Args& a, int tile, int bm, int lane, int& lo, int& hi) {
    int before = 0;
    for (int e0 = 0; e0 < a.E; e0 += 64) {
        const int e = e0 + lane;
        Span s{0, 0};
        if (e < a.E) s = span_of(a.offsets, e, a.T);
        const int n = (s.hi - s.lo + bm - 1) / bm;
        int sum = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int up = __shfl_up(sum, o, 64);
            if (lane >= o) sum += up;
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
    if (a.zero_rest) {
        int end = a.offsets[a.E];
        end = end < 0 ? 0 : (end > a.T ? a.T : end);
        lo = end + (tile - before) * bm;
        hi = min(a.T, lo + bm);
        if (lo < hi) return a.E;
    }
    return -1;
}

__device__ __forceinline__ int kmaj_key(int kr) { return ((kr >> 1) & 1) | (((kr >> 3) & 1) << 1); }

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
        const char* base = u + kq * 128 + (((f & 3) ^ kmaj_key(kq)) << 5) + (p << 3);
        const bf16x4 lo = lds_read_tr_raw(base, s * 4096), hi = lds_read_tr_raw(base, s * 4096 + 512);
        return cat8(lo, hi);
    }
}

enum { FWD = 0, DX = 1, DW = 2 };

// BM x BN tile, four waves of (BM / 2) x (BN / 2), two LDS stages of 64 reduction steps.
template <int WHAT, int BM, int BN>
__global__ __launch_bounds__(THREADS, 2) void grouped_kernel(Args a, int tiles_j, int tiles_i) {
    constexpr bool XK = WHAT == DW, YK = WHAT != FWD;
    constexpr int UX = BM / 64, UY = BN / 64, FM = BM / 32, FN = BN / 32, STAGE = (UX + UY) * UNIT;
    __shared__ __attribute__((aligned(16))) char lds[2][STAGE];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1, g = lane >> 4, li = lane & 15;
    int work = xcd_remap(blockIdx.x, gridDim.x);
    int e, lo, hi, i0, j0, k_end, kt0 = 0, kt1, slice = 0;
    if constexpr (WHAT == DW) {
        const int per = tiles_i * tiles_j;
        slice = work % a.slices;
        work /= a.slices;
        e = work / per;
        i0 = (work % per) / tiles_j * BM;
        j0 = work % tiles_j * BN;
        const Span s = span_of(a.offsets, e, a.T);
        lo = s.lo;
        hi = s.hi;
        k_end = hi - lo;
        const int nk_all = (k_end + BK - 1) / BK, each = (nk_all + a.slices - 1) / a.slices;
        kt0 = min(slice * each, nk_all);
        kt1 = min(kt0 + each, nk_all);
    } else {
        e = find_tile(a, work / tiles_j, BM, lane, lo, hi);
        if (e < 0) return;
        i0 = 0;
        j0 = work % tiles_j * BN;
        k_end = e == a.E ? 0 : (WHAT == FWD ? a.K : a.N);
        kt1 = (k_end + BK - 1) / BK;
    }
    const int nk = kt1 - kt0;
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

    if (nk > 0) {
        // a lane's place in a unit: row (or reduction step) r0 and r0 + 32, sixteen bytes at column c
        const int r0 = tid >> 3;
        const int cc = ((tid & 7) ^ (r0 & 7)) * 8;                                            // k-contiguous
        const int ck = ((((tid & 7) >> 1) ^ kmaj_key(r0)) * 2 + (tid & 1)) * 8;               // k-major
        const bf16* wbase = WHAT == DW ? nullptr : a.w + (long)e * a.stride_w;
        const bf16* xrow[XK ? 1 : UX][2];
        if constexpr (!XK) {
            const bf16* src = WHAT == FWD ? a.x : a.dy;
            const long ld = WHAT == FWD ? a.ldx : a.ldy;
#pragma unroll
            for (int u = 0; u < UX; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    int i = lo + u * 64 + h * 32 + r0;
                    i = i < hi ? i : hi - 1;                       // rows behind the tile's last feed results nobody stores
                    int row = a.rows ? a.rows[i] : i;
                    row = (unsigned)row < (unsigned)a.T ? row : 0;
                    xrow[u][h] = src + row * ld + cc;
                }
        }
        auto stage = [&](int kt, int st) {
            char* dst = lds[st] + wave * 1024;
            const int k0 = kt * BK;
            if constexpr (WHAT == DW) {
                long row[2];
                bool in[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int k = k0 + h * 32 + r0;
                    in[h] = k < k_end;
                    const int i = lo + (in[h] ? k : 0);
                    const int r = a.rows ? a.rows[i] : i;
                    in[h] = in[h] && (unsigned)r < (unsigned)a.T;
                    row[h] = in[h] ? r : 0;
                }
#pragma unroll
                for (int u = 0; u < UX + UY; ++u) {
                    const bool isx = u < UX;
                    const int ext = isx ? a.N : a.K;
                    int col = (isx ? i0 + u * 64 : j0 + (u - UX) * 64) + ck;
                    col = col <= ext - 8 ? col : ext - 8;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const bf16* p = isx ? a.dy + row[h] * a.ldy + col : a.x + row[h] * a.ldx + col;
                        dma16(in[h] ? (const void*)p : (const void*)kZeros, dst + u * UNIT + h * 4096);
                    }
                }
            } else {
#pragma unroll
                for (int u = 0; u < UX; ++u)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        dma16(k0 + cc < k_end ? (const void*)(xrow[u][h] + k0) : (const void*)kZeros, dst + u * UNIT + h * 4096);
#pragma unroll
                for (int u = 0; u < UY; ++u)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const void* p;
                        if constexpr (YK) {
                            const int k = k0 + h * 32 + r0;
                            int col = j0 + u * 64 + ck;
                            col = col <= NJ - 8 ? col : NJ - 8;
                            p = k < k_end ? (const void*)(wbase + k * a.ldw + col) : (const void*)kZeros;
                        } else {
                            int j = j0 + u * 64 + h * 32 + r0;
                            j = j < NJ ? j : NJ - 1;
                            p = k0 + cc < k_end ? (const void*)(wbase + j * a.ldw + k0 + cc) : (const void*)kZeros;
                        }
                        dma16(p, dst + (UX + u) * UNIT + h * 4096);
                    }
            }
        };
        stage(kt0, 0);
        const bf16x8 ones = {(bf16)1.f, (bf16)1.f, (bf16)1.f, (bf16)1.f, (bf16)1.f, (bf16)1.f, (bf16)1.f, (bf16)1.f};
#pragma unroll 1
        for (int t = 0; t < nk; ++t) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();                                         // stage t & 1 is complete, the other one is free
            if (t + 1 < nk) stage(kt0 + t + 1, (t + 1) & 1);
            const char* lx = lds[t & 1];
            const char* ly = lds[t & 1] + UX * UNIT;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                bf16x8 xf[FM], yf[FN];
#pragma unroll
                for (int m = 0; m < FM; ++m) xf[m] = frag<XK>(lx, wm * FM + m, s, lane);
#pragma unroll
                for (int n = 0; n < FN; ++n) yf[n] = frag<YK>(ly, wn * FN + n, s, lane);
                if constexpr (XK) lds_fence(xf);
                if constexpr (YK) lds_fence(yf);
#pragma unroll
                for (int m = 0; m < FM; ++m)
#pragma unroll
                    for (int n = 0; n < FN; ++n)
                        acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(yf[n], xf[m], acc[m][n], 0, 0, 0);
                if constexpr (WHAT == DW) {
                    if (sums) {
#pragma unroll
                        for (int m = 0; m < FM; ++m) rs[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, xf[m], rs[m], 0, 0, 0);
                    }
                }
            }
        }
    }
    // a lane holds C[row li of fragment m][4 g .. 4 g + 3 of fragment n]
    if constexpr (WHAT == DW) {
        const long plane = (long)a.N * a.K;
        float* out = a.dw + ((long)slice * a.E + e) * plane;
#pragma unroll
        for (int m = 0; m < FM; ++m) {
            const int i = i0 + (wm * FM + m) * 16 + li;
#pragma unroll
            for (int n = 0; n < FN; ++n) {
                const int j = j0 + (wn * FN + n) * 16 + g * 4;
                if (i < a.N && j < a.K) *reinterpret_cast<f32x4*>(out + (long)i * a.K + j) = acc[m][n];
            }
            if (sums && g == 0 && i < a.N) a.db[((long)slice * a.E + e) * a.N + i] = rs[m][0];
        }
    } else {
        const float* bias = WHAT == FWD && a.bias && e < a.E ? a.bias + (long)e * a.stride_b : nullptr;
        f32x4 bv[FN];
#pragma unroll
        for (int n = 0; n < FN; ++n) {
            const int j = j0 + (wn * FN + n) * 16 + g * 4;
            bv[n] = bias && j < NJ ? *reinterpret_cast<const f32x4*>(bias + j) : f32x4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int m = 0; m < FM; ++m) {
            const int i = lo + (wm * FM + m) * 16 + li;
            int row = i < hi ? (a.rows ? a.rows[i] : i) : -1;
            if ((unsigned)row >= (unsigned)a.T) continue;
            bf16* out = (bf16*)a.out + row * a.ldo;
#pragma unroll
            for (int n = 0; n < FN; ++n) {
                const int j = j0 + (wn * FN + n) * 16 + g * 4;
                const f32x4 v = acc[m][n] + bv[n];
                if (j < NJ) *reinterpret_cast<bf16x4*>(out + j) = pack4(v[0], v[1], v[2], v[3]);
            }
        }
    }
}

// out[i] = sum over the slices of dW / db, in order
__global__ __launch_bounds__(256) void slice_sum_kernel(const float* __restrict__ part, float* __restrict__ out, long n4,
                                                        int slices) {
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n4; i += (long)gridDim.x * 256) {
        f32x4 v = reinterpret_cast<const f32x4*>(part)[i];
        for (int s = 1; s < slices; ++s) v += reinterpret_cast<const f32x4*>(part)[s * n4 + i];
        reinterpret_cast<f32x4*>(out)[i] = v;
    }
}

// ------------------------------------------------------------------ rows in the order of their experts
constexpr int SORT_THREADS = 1024, SORT_WAVES = 16, SORT_MAX_E = 512;

__device__ __forceinline__ int key_of(const int* expert, int t, int T, int E) {
    const int e = t < T ? expert[t] : E;
    return (unsigned)e < (unsigned)E ? e : E;
}

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
// after a scan over (key, wave) -- writing.  Keys are experts, E for a row that none takes.
__global__ __launch_bounds__(SORT_THREADS) void expert_rows_kernel(const int* __restrict__ expert, int T, int E, int bits,
                                                                   int* __restrict__ rows, int* __restrict__ offsets) {
    __shared__ int count[SORT_WAVES][SORT_MAX_E + 1];
    __shared__ int wave_total[SORT_WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, keys = E + 1;
    for (int i = tid; i < SORT_WAVES * keys; i += SORT_THREADS) count[i / keys][i % keys] = 0;
    __syncthreads();
    const int chunks = (T + 63) / 64, each = (chunks + SORT_WAVES - 1) / SORT_WAVES;
    const int c0 = wave * each, c1 = min(c0 + each, chunks);
    for (int c = c0; c < c1; ++c) {
        const int t = c * 64 + lane;
        const int key = key_of(expert, t, T, E);
        const bool in = t < T;
        const unsigned long long live = __ballot(in), mask = same_key(key, bits) & live;
        if (in && lane == __builtin_ctzll(mask)) count[wave][key] += __popcll(mask);
    }
    __syncthreads();
    // exclusive scan in the order (key, wave): thread k owns key k
    int mine = 0;
    if (tid < keys)
        for (int w = 0; w < SORT_WAVES; ++w) mine += count[w][tid];
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(sum, o, 64);
        if (lane >= o) sum += up;
    }
    if (lane == 63) wave_total[wave] = sum;
    __syncthreads();
    int base = sum - mine;
    for (int w = 0; w < wave; ++w) base += wave_total[w];
    if (tid < keys) {
        offsets[tid] = base;                       // key E: the end of the last expert's rows
        for (int w = 0; w < SORT_WAVES; ++w) {
            const int n = count[w][tid];
            count[w][tid] = base;
            base += n;
        }
    }
    __syncthreads();
    for (int c = c0; c < c1; ++c) {
        const int t = c * 64 + lane;
        const int key = key_of(expert, t, T, E);
        const bool in = t < T;
        const unsigned long long live = __ballot(in), mask = same_key(key, bits) & live;
        if (in) {
            const int first = __builtin_ctzll(mask);
            const int at = count[wave][key];       // every lane of the key reads before its first lane moves it on
            rows[at + __popcll(mask & ((1ull << lane) - 1))] = t;
            if (lane == first) count[wave][key] = at + __popcll(mask);
        }
    }
}

int cdiv(long a, long b) { return (int)((a + b - 1) / b); }

}  // namespace

extern "C" int vp_expert_rows(const int* expert, int T, int E, int* rows, int* offsets, hipStream_t stream) {
    VP_CHECK_ARG(T >= 0 && E >= 1 && offsets && (T == 0 || (expert && rows)));
    if (E > SORT_MAX_E) return VP_ERR_UNSUPPORTED;
    int bits = 1;
    while ((1 << bits) <= E) ++bits;
    hipLaunchKernelGGL(expert_rows_kernel, dim3(1), dim3(SORT_THREADS), 0, stream, expert, T, E, bits, rows, offsets);
    VP_LAUNCH_RET();
}

namespace {

int check_common(const vp_grouped_args* g) {
    VP_CHECK_ARG(g && g->T >= 0 && g->E >= 1 && g->N >= 8 && g->K >= 8 && g->N % 8 == 0 && g->K % 8 == 0 && g->offsets);
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

// upper bound of the row tiles: every expert's last tile may be partial; rows behind the last expert add one more
int row_tiles(const vp_grouped_args* g, int bm) {
    const long groups = (long)g->E < g->T ? g->E : g->T;
    return (int)(g->T / bm + groups + (g->zero_rest ? 1 : 0));
}

template <int WHAT>
int launch_rows(const vp_grouped_args* g, hipStream_t stream) {
    const Args a = make_args(g);
    const int nj = WHAT == FWD ? g->N : g->K;
    constexpr int BM = 128, BN = 128;
    const int tj = cdiv(nj, BN);
    const long grid = (long)row_tiles(g, BM) * tj;
    VP_CHECK_ARG(grid <= 0x7FFFFFFF);
    hipLaunchKernelGGL((grouped_kernel<WHAT, BM, BN>), dim3((unsigned)grid), dim3(THREADS), 0, stream, a, tj, 0);
    VP_LAUNCH_RET();
}

int dw_slices(int T, int E, int N, int K) {
    const long tiles = (long)E * cdiv(N, 128) * cdiv(K, 128);
    long s = 512 / (tiles < 1 ? 1 : tiles);
    const long most = (T + 511) / 512;
    s = s > most ? most : s;
    return s < 1 ? 1 : (int)s;
}

}  // namespace

extern "C" int vp_grouped_fwd(const vp_grouped_args* g, hipStream_t stream) {
    if (int rc = check_common(g)) return rc;
    if (g->T == 0) return VP_OK;
    VP_CHECK_ARG(g->x && g->w && g->out && aligned16(g->x) && aligned16(g->w) && aligned16(g->out));
    VP_CHECK_ARG(g->ldx >= g->K && g->ldw >= g->K && g->ldo >= g->N && g->ldx % 8 == 0 && g->ldw % 8 == 0 && g->ldo % 8 == 0);
    VP_CHECK_ARG(g->stride_w % 8 == 0 && (!g->bias || (aligned16(g->bias) && g->stride_b % 4 == 0)));
    return launch_rows<FWD>(g, stream);
}

extern "C" int vp_grouped_dgrad(const vp_grouped_args* g, hipStream_t stream) {
    if (int rc = check_common(g)) return rc;
    if (g->T == 0) return VP_OK;
    VP_CHECK_ARG(g->dy && g->w && g->out && aligned16(g->dy) && aligned16(g->w) && aligned16(g->out));
    VP_CHECK_ARG(g->ldy >= g->N && g->ldw >= g->K && g->ldo >= g->K && g->ldy % 8 == 0 && g->ldw % 8 == 0 && g->ldo % 8 == 0);
    VP_CHECK_ARG(g->stride_w % 8 == 0);
    return launch_rows<DX>(g, stream);
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
    const int ti = cdiv(g->N, 128), tj = cdiv(g->K, 128);
    a.slices = dw_slices(g->T, g->E, g->N, g->K);
    const size_t need = a.slices == 1 ? 0 : (size_t)a.slices * g->E * g->N * ((size_t)g->K + (db ? 1 : 0)) * 4;
    VP_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && aligned16(workspace)));
    const long n = (long)g->E * g->N * g->K, nb = (long)g->E * g->N;
    a.dw = a.slices == 1 ? dw : (float*)workspace;
    a.db = a.slices == 1 ? db : (db ? (float*)workspace + a.slices * n : nullptr);
    const long grid = (long)g->E * ti * tj * a.slices;
    VP_CHECK_ARG(grid <= 0x7FFFFFFF);
    hipLaunchKernelGGL((grouped_kernel<DW, 128, 128>), dim3((unsigned)grid), dim3(THREADS), 0, stream, a, tj, ti);
    if (a.slices > 1) {
        const int blocks = (int)(n / 4 < 2048L * 256 ? cdiv(n / 4, 256) : 2048);
        hipLaunchKernelGGL(slice_sum_kernel, dim3(blocks), dim3(256), 0, stream, a.dw, dw, n / 4, a.slices);
        if (db)
            hipLaunchKernelGGL(slice_sum_kernel, dim3(cdiv(nb / 4, 256)), dim3(256), 0, stream, a.db, db, nb / 4, a.slices);
    }
    VP_LAUNCH_RET();
}
