// A linear layer over the rows of many sequences with a low-rank adapter per sequence beside the shared weight:
//   y_n = act(W x_n + b + scale_a Up_a (Down_a x_n)),   a = ids[sequence of n]   (negative: the shared layer alone).
// Two launches: z = scale Down x for all rows (mp_adapt_down, fp32 into the workspace), then the shared product with Up z joined
// to it in its registers before the one rounding and the one store (mp_adapt_gemm).  Up to three operands of a product decide the arithmetic:
// bf16 inputs go to the bf16 matrix instructions as they are; fp32 inputs as three bf16 terms each (hi + mid + lo, each the nearest
// to what is left: all 24 bits), six products per fp32 product -- the three left out are below 2^-26 of it --, fp32 accumulation:
// the accuracy of an fp32 sum at 16 / 6 times the rate of the fp32 matrix instructions.  (An infinite fp32 input gives NaN:
// inf - inf in the split.)
#include "mp_seq_dev.h"

namespace mpseq {

size_t adapt_ws_floats(int B, int T, int r) { return (size_t)B * T * r; }

// ---------------------------------------------------------------- z = scale Down x
// A workgroup takes up to 16 frames of one sequence -- one adapter, so the product runs on the matrix units even where the 16 rows
// are one (a tick: the reads of Down bound it either way) --, K split over the four waves and joined through LDS.
template <class E>
MP_KERNEL __launch_bounds__(256) void mp_adapt_down(AdaptArgs a, int per_seq) {
    constexpr int P = Arith<E>::P;
    __shared__ float part[4][16][17];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, grp = lane >> 4;
    const int b = blockIdx.x / per_seq, t0 = blockIdx.x % per_seq * 16, id = a.ids[b];
    if (id < 0 || id >= a.n) return;                              // (the second launch reads no z of such rows)
    const int t = t0 + col < a.T ? t0 + col : a.T - 1;
    const E* x = (const E*)a.x + (size_t)b * a.sx[0] + (size_t)t * a.sx[1];
    const float sc = a.scale ? a.scale[id] : 1.f;
    for (int j0 = 0; j0 < a.r; j0 += 16) {
        const int j = j0 + col < a.r ? j0 + col : a.r - 1;
        const E* d = (const E*)a.down + ((size_t)id * a.r + j) * a.K;
        f32x4 acc = {};
        int k = (wave * 4 + grp) * 8;
#pragma unroll 2
        for (; k - grp * 8 + 32 <= a.K; k += 128) {
            Oct<E> ox, od;
            u32x4 px[P], pd[P];
            ox.load(x + k); od.load(d + k);
            ox.planes(px); od.planes(pd);
            acc = mfma_planes(pd, px, acc);
        }
        if (k - grp * 8 < a.K) {
            const int left = a.K - k < 0 ? 0 : a.K - k;
            Oct<E> ox, od;
            u32x4 px[P], pd[P];
            ox.load_some(x + k, left); od.load_some(d + k, left);
            ox.planes(px); od.planes(pd);
            acc = mfma_planes(pd, px, acc);
        }
        for (int r = 0; r < 4; ++r) part[wave][4 * grp + r][col] = acc[r];      // [component][row]
        __syncthreads();
        const int row = tid >> 4, c = tid & 15;
        if (t0 + row < a.T && j0 + c < a.r)
            a.ws[((size_t)b * a.T + t0 + row) * a.r + j0 + c] = sc * ((part[0][c][row] + part[1][c][row]) + (part[2][c][row] + part[3][c][row]));
        __syncthreads();
    }
}

// ---------------------------------------------------------------- the shared product, the adapters' second half joined to it
// A workgroup's tile is (32 MR rows of x) x (32 MC columns of y); four waves, 2 x 2, each MR x MC tiles of 16 x 16 with W as the A
// operand (so that a lane ends with four consecutive columns of one row).  Tiles of K go through registers into LDS, rows padded by
// 16 bytes (a 16-lane read of one K group covers every bank once); the next tile's loads are in flight while this one is
// multiplied.
template <class E, int MR, int MC>
MP_KERNEL __launch_bounds__(256) void mp_adapt_gemm(AdaptArgs a, int rows, int ntr, int ntc) {
    constexpr int P = Arith<E>::P, BK = P == 1 ? 64 : 32, UR = BK / 8, RN = 32 * MR, CM = 32 * MC, LS = BK + 8;
    constexpr int NU = (RN + CM) * UR / 256;                      // units of eight elements that a thread stages
    static_assert((RN + CM) * UR % 256 == 0, "whole units per thread");
    __shared__ __align__(16) bf16raw lds[P][RN + CM][LS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, grp = lane >> 4;
    // workgroups are dealt to the 8 XCDs in turn: a run of tiles (columns fastest: one panel of x) to each, so that an XCD's L2
    // holds what its tiles share
    const int nt = ntr * ntc, per = (nt + 7) / 8, tile = (int)(blockIdx.x % 8) * per + (int)(blockIdx.x / 8);
    if (tile >= nt || (int)(blockIdx.x / 8) >= per) return;
    const int n0 = tile / ntc * RN, m0 = tile % ntc * CM;
    const E* src[NU];
#pragma unroll
    for (int u = 0; u < NU; ++u) {
        const int row = (tid + 256 * u) / UR, kk = (tid + 256 * u) % UR * 8;
        if (row < RN) {
            const int n = n0 + row < rows ? n0 + row : rows - 1, b = n / a.T;
            src[u] = (const E*)a.x + (size_t)b * a.sx[0] + (size_t)(n - b * a.T) * a.sx[1] + kk;
        } else {
            const int m = m0 + row - RN < a.M ? m0 + row - RN : a.M - 1;
            src[u] = (const E*)a.w + (size_t)m * a.K + kk;
        }
    }
    const int wr = wave & 1, wc = wave >> 1;
    f32x4 acc[MC][MR] = {};
    Oct<E> oct[NU];
    auto fetch = [&](int k0) {
        if (k0 + BK <= a.K) {
#pragma unroll
            for (int u = 0; u < NU; ++u) oct[u].load(src[u] + k0);
        } else {
#pragma unroll
            for (int u = 0; u < NU; ++u) oct[u].load_guarded(src[u] + k0, a.K - k0 - (tid + 256 * u) % UR * 8);
        }
    };
    fetch(0);
    for (int k0 = 0; k0 < a.K; k0 += BK) {
        __syncthreads();
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const int row = (tid + 256 * u) / UR, kk = (tid + 256 * u) % UR * 8;
            u32x4 p[P];
            oct[u].planes(p);
#pragma unroll
            for (int i = 0; i < P; ++i) *(u32x4*)&lds[i][row][kk] = p[i];
        }
        __syncthreads();
        if (k0 + BK < a.K) fetch(k0 + BK);
#pragma unroll
        for (int ks = 0; ks < BK; ks += 32) {
            u32x4 fx[MR][P];
#pragma unroll
            for (int i = 0; i < MR; ++i)
#pragma unroll
                for (int p = 0; p < P; ++p) fx[i][p] = *(const u32x4*)&lds[p][(wr * MR + i) * 16 + col][ks + 8 * grp];
#pragma unroll
            for (int j = 0; j < MC; ++j) {
                u32x4 fw[P];
#pragma unroll
                for (int p = 0; p < P; ++p) fw[p] = *(const u32x4*)&lds[p][RN + (wc * MC + j) * 16 + col][ks + 8 * grp];
#pragma unroll
                for (int i = 0; i < MR; ++i) acc[j][i] = mfma_planes(fw, fx[i], acc[j][i]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MR; ++i) {
        const int nb = n0 + (wr * MR + i) * 16;                   // 16 rows, one per lane column
        const int n = nb + col, nc = n < rows ? n : rows - 1;
        const int id = a.ids[nc / a.T];
        const bool use = id >= 0 && id < a.n;
        const float* z = a.ws + (size_t)nc * a.r;
        const int id0 = __builtin_amdgcn_readfirstlane(id);
        if (__all(id == id0)) {
            if (id0 >= 0 && id0 < a.n)                            // one adapter for the 16 rows: the matrix units again
                for (int r0 = 0; r0 < a.r; r0 += 32) {
                    const int k = r0 + 8 * grp, left = a.r - k < 0 ? 0 : a.r - k;
                    Oct<float> oz;
                    u32x4 p3[3], pz[P == 1 ? 2 : 3];              // z keeps 16 of its bits beside bf16 operands, all 24 beside fp32 ones
                    oz.load_some(z + k, left);
                    oz.planes(p3);
#pragma unroll
                    for (int p = 0; p < (P == 1 ? 2 : 3); ++p) pz[p] = p3[p];
#pragma unroll
                    for (int j = 0; j < MC; ++j) {
                        const int m = m0 + (wc * MC + j) * 16 + col;
                        Oct<E> ou;
                        u32x4 pu[P];
                        ou.load_some((const E*)a.up + ((size_t)id0 * a.M + (m < a.M ? m : 0)) * a.r + k, left);
                        ou.planes(pu);
                        acc[j][i] = mfma_planes(pu, pz, acc[j][i]);
                    }
                }
        } else if (use) {                                         // a row of its own each: dot products of the lane's four columns
            for (int q = 0; q < a.r; q += 8) {
                Oct<float> oz;
                oz.load_some(z + q, a.r - q);
#pragma unroll
                for (int j = 0; j < MC; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int m = m0 + (wc * MC + j) * 16 + 4 * grp + r;
                        Oct<E> ou;
                        ou.load_some((const E*)a.up + ((size_t)id * a.M + (m < a.M ? m : 0)) * a.r + q, a.r - q);
                        acc[j][i][r] = ou.dot(oz, acc[j][i][r]);
                    }
            }
        }
        if (n >= rows) continue;
#pragma unroll
        for (int j = 0; j < MC; ++j) {
            const int m = m0 + (wc * MC + j) * 16 + 4 * grp;
            float y[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                y[r] = acc[j][i][r] + (a.bias && m + r < a.M ? load_f((const E*)a.bias + m + r) : 0.f);
                if (id >= a.n) y[r] = __builtin_nanf("");
                if (a.relu) y[r] = relu_(y[r]);
            }
            E* out = (E*)a.y + (size_t)n * a.M + m;
            if (a.vec) {                                          // M a multiple of 4: whole groups of columns, aligned
                if (m < a.M) store4(out, y);
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (m + r < a.M) store_f(out + r, y[r]);
            }
        }
    }
}

template <class E, int MR, int MC>
static void gemm_for(const AdaptArgs& a, int rows, hipStream_t s) {
    const int ntr = (rows + 32 * MR - 1) / (32 * MR), ntc = (a.M + 32 * MC - 1) / (32 * MC);
    hipLaunchKernelGGL((mp_adapt_gemm<E, MR, MC>), dim3((unsigned)((ntr * ntc + 7) / 8 * 8)), dim3(256), 0, s, a, rows, ntr, ntc);
}
template <class E>
static bool launch_for(AdaptArgs a, hipStream_t s) {
    const int rows = a.B * a.T;
    a.vec = a.M % 4 == 0 && (uintptr_t)a.y % (4 * sizeof(E)) == 0;
    hipLaunchKernelGGL(mp_adapt_down<E>, dim3((unsigned)(a.B * ((a.T + 15) / 16))), dim3(256), 0, s, a, (a.T + 15) / 16);
    auto tiles = [&](int t) { return ((long)rows + t - 1) / t * ((a.M + t - 1) / t); };
    if (tiles(128) >= 192) gemm_for<E, 4, 4>(a, rows, s);
    else if (tiles(64) >= 192) gemm_for<E, 2, 2>(a, rows, s);
    else gemm_for<E, 1, 1>(a, rows, s);
    return hipGetLastError() == hipSuccess;
}
bool launch_adapt(const AdaptArgs& a, int dtype, hipStream_t s) {
    return dtype == kBF16 ? launch_for<bf16raw>(a, s) : launch_for<float>(a, s);
}

}  // namespace mpseq
