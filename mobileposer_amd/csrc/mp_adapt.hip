// A linear layer over the rows of many sequences with a low-rank adapter per sequence beside the shared weight:
//   y_n = act(W x_n + b + scale_a Up_a (Down_a x_n)),   a = ids[sequence of n]   (negative: the shared layer alone).
// Wide layers take two launches: z = scale Down x for all rows (mp_adapt_down, fp32 into the workspace), then the shared product with
// Up z joined to it in its registers before the one rounding and the one store (mp_adapt_gemm).  Where a layer's columns and
// the adapter's components fit one tile side by side (an output layer) and the sequences are long, Down's rows ride in the shared
// product as further columns and x is read once (mp_adapt_gemm<.., FUSED>).
// bf16 inputs go to the bf16 matrix instructions as they are, fp32 inputs as three bf16 terms each (mp_seq_dev.h).  Terms hold no
// infinity, nor the last half step of bf16 below FLT_MAX (the first term would be infinite, the next ones NaN): a result that is not finite is
// computed again from the inputs in fp32 (plain_dot, plain_tile).  That keeps infinities what they are in an fp32 product.  It costs a
// look at every result: no time that can be measured; with one infinite sample 8 x 2048 (2048 -> 2048, bf16) 149 -> 302 us, with nothing
// but NaN 5.7 ms.
#include "mp_seq_dev.h"

#include <utility>

namespace mpseq {

size_t adapt_ws_floats(int B, int T, int r) { return (size_t)B * T * r; }
// 32-bit row and z indexes; workgroups of up to 512 threads in a launch that counts its threads in 32 bits: one per 16 frames of a
// sequence (Down), one per 128 of them (one launch), tiles of 128 or 256 from 192 or 384 of 128 on (the smaller tiles in front of that
// are a few thousand)
bool adapt_fits(int B, int T, int M, int r) {
    const int64_t rows = (int64_t)B * T, most = (1 << 23) - 8;
    return rows <= 1 << 30 && rows * r <= 0x7fffffff && (int64_t)B * ((T + 15) / 16) <= most && (rows + 127) / 128 * (((int64_t)M + 127) / 128) <= most;
}

static __device__ __forceinline__ bool not_finite(float x) { return !(fabsf(x) <= 3.402823466e38f); }
template <class E>
static __device__ __forceinline__ const E* row_of_x(const AdaptArgs& a, int n) {
    const int b = n / a.T;
    return (const E*)a.x + (size_t)b * a.sx[0] + (size_t)(n - b * a.T) * a.sx[1];
}
template <class E>
static __device__ __forceinline__ float plain_dot(const E* x, const E* w, int K) {
    float s = 0.f;
    for (int k = 0; k < K; ++k) s = fmaf(load_f(x + k), load_f(w + k), s);
    return s;
}

// ---------------------------------------------------------------- z = scale Down x
// A workgroup takes up to 16 RG frames of one sequence -- one adapter, so the product runs on the matrix units even where the rows
// are one (a tick: the reads of Down bound it either way) --, K split over the four waves and joined through LDS; KB steps of
// every wave are in flight together.  RT = r / 16 rounded up.  Bound by the latency of one pass for a tick (512 x 1, 1024, r 16: 6 us), by
// the reads of x and Down together for long sequences (8 x 2048, 2048, r 32: 18 .. 20 us, 67 MB of x and as many of Down, those from L2).
template <class E, int RT, int RG>
MP_KERNEL __launch_bounds__(256) void mp_adapt_down(AdaptArgs a, int per_seq) {
    constexpr int P = Arith<E>::P, KB = RT >= 4 ? 2 : 4, NR = 16 * RG;
    __shared__ float part[4][16 * RT][NR + 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, grp = lane >> 4;
    const int b = blockIdx.x / per_seq, t0 = blockIdx.x % per_seq * NR, id = a.ids[b];
    if (id < 0 || id >= a.n) return;                              // (the second launch reads no z of such rows)
    const E* x[RG];
#pragma unroll
    for (int g = 0; g < RG; ++g) x[g] = (const E*)a.x + (size_t)b * a.sx[0] + (size_t)min(t0 + 16 * g + col, a.T - 1) * a.sx[1];
    const E* d[RT];
#pragma unroll
    for (int j = 0; j < RT; ++j) d[j] = (const E*)a.down + ((size_t)id * a.r + min(16 * j + col, a.r - 1)) * a.K;
    f32x4 acc[RG][RT] = {};
    int k = (wave * 4 + grp) * 8;
    for (; k - grp * 8 + 128 * (KB - 1) + 32 <= a.K; k += 128 * KB) {
        Oct<E> ox[KB][RG], od[KB][RT];
#pragma unroll
        for (int m = 0; m < KB; ++m) {
#pragma unroll
            for (int g = 0; g < RG; ++g) ox[m][g].load(x[g] + k + 128 * m);
#pragma unroll
            for (int j = 0; j < RT; ++j) od[m][j].load(d[j] + k + 128 * m);
        }
#pragma unroll
        for (int m = 0; m < KB; ++m) {
            u32x4 px[P], pd[RT][P];
#pragma unroll
            for (int j = 0; j < RT; ++j) od[m][j].planes(pd[j]);
#pragma unroll
            for (int g = 0; g < RG; ++g) {
                ox[m][g].planes(px);
                mfma_planes_n<RT, P, P>(pd, px, acc[g]);
            }
        }
    }
    for (; k - grp * 8 < a.K; k += 128) {
        const int left = a.K - k < 0 ? 0 : a.K - k;
        Oct<E> ox, od;
        u32x4 px[P], pd[RT][P];
#pragma unroll
        for (int j = 0; j < RT; ++j) {
            od.load_some(d[j] + k, left);
            od.planes(pd[j]);
        }
#pragma unroll
        for (int g = 0; g < RG; ++g) {
            ox.load_some(x[g] + k, left);
            ox.planes(px);
            mfma_planes_n<RT, P, P>(pd, px, acc[g]);
        }
    }
#pragma unroll
    for (int g = 0; g < RG; ++g)
#pragma unroll
        for (int j = 0; j < RT; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) part[wave][16 * j + 4 * grp + r][16 * g + col] = acc[g][j][r];      // [component][row]
    __syncthreads();
    const float sc = a.scale ? a.scale[id] : 1.f;
    for (int i = tid; i < NR * a.r; i += 256) {
        const int row = i / a.r, c = i % a.r;
        if (t0 + row < a.T) {
            float z = (part[0][c][row] + part[1][c][row]) + (part[2][c][row] + part[3][c][row]);
            if (P > 1 && not_finite(z)) z = plain_dot(row_of_x<E>(a, b * a.T + t0 + row), (const E*)a.down + ((size_t)id * a.r + c) * a.K, a.K);
            a.ws[((size_t)b * a.T + t0 + row) * a.r + c] = sc * z;
        }
    }
}

// ---------------------------------------------------------------- the shared product, the adapters' second half joined to it
// A workgroup's tile is RN rows of x times CM columns of y; WR x WC waves, each MR x MC tiles of 16 x 16 with W as the A operand (so
// that a lane ends with four consecutive columns of one row).  Tiles of BK along K go through registers into LDS -- consecutive lanes
// load consecutive pieces of a row: a wave's loads are whole cache lines, which is what bounds it otherwise -- as blocks of 16
// rows x 32 in operand order, the 16-byte pieces of a block exchanged by block_piece() so that neither side meets a bank more
// than twice.  (Any order of K serves that all operands share: an fp32 piece is two runs of four, half a tile apart, so that a
// load of 16 bytes a lane has no gaps between the lanes either.)  The next tile's loads are in flight while this one is
// multiplied.  BK is as long as the staging registers allow: a small tile is a chain of memory latencies.  FUSED: a row tile lies
// inside one sequence, columns Mp .. Mp + r - 1 of the tile (Mp = M rounded up to 16) are that sequence's Down.  DIRECT (bf16, rows of
// whole cache lines): tiles go from memory to LDS without registers, 8 rows x 128 bytes a wave and instruction, the pieces of a row
// exchanged by its index; the fragments are read between the products.  8 x 2048, 2048 -> 2048, r 32: 126 .. 137 us, 1090 .. 1000 TFLOP/s (the
// library's product: 1180), 1.35 us per step of K beside 0.85 of products alone, 18 us for loads before and stores behind;
// 256 x 125, 512 -> 96, r 8, fp32 (FUSED): 29 us, 2.8 TB/s, 1.4 us per step of K beside 0.64 of products alone (LDS and splitting the rest).
template <class E, int WR, int WC, int MR, int MC, int BK, bool TWO, bool FUSED, bool DIRECT>
struct Gemm {
    static constexpr int P = Arith<E>::P, KS = BK / 32, RN = 16 * MR * WR, CM = 16 * MC * WC, TH = 64 * WR * WC;
    static constexpr int UR = BK / 8, NB = (RN + CM) / 16 * KS, NU = (RN + CM) * UR / TH;      // blocks of a tile; pieces that a thread stages
    static constexpr int kPlane = NB * 1024, kOne = P * kPlane, kZ = TWO ? 2 * kOne : kOne, kRowZ = 128 + 4;
    static constexpr bool kTurn = !FUSED && 16 * MC * sizeof(E) >= 128 && RN * CM * (int)sizeof(E) <= kZ;      // outputs leave through LDS
    static constexpr int kBytes = FUSED ? (kZ > RN * kRowZ * 4 ? kZ : RN * kRowZ * 4) : kZ;      // (z takes the operands' place)
    static_assert((RN + CM) * UR % TH == 0 && kBytes <= 160 * 1024, "whole pieces per thread, LDS of a CU");
};
// Outputs of rows n .. n + 15 and columns m .. m + 15 that are not finite, from the inputs on the fp32 matrix instructions (a wave; z: of
// the lane's row n + lane % 16)
template <class E>
static __device__ __forceinline__ void plain_tile(const AdaptArgs& a, int n, int n1, int m, const float* z) {
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4, row = min(n + col, n1 - 1), b = row / a.T, id = a.ids[b];
    E* const y = (E*)a.y + (size_t)b * a.sy[0] + (size_t)(row - b * a.T) * a.sy[1];
    bool odd[4], any = false;
    for (int r = 0; r < 4; ++r) {
        const int c = m + 4 * grp + r;
        odd[r] = n + col < n1 && c < a.M && id < a.n && not_finite(load_f(y + min(c, a.M - 1)));
        any = any || odd[r];
    }
    if (!__any(any)) return;
    const E* x = row_of_x<E>(a, row);
    const E* w = (const E*)a.w + (size_t)min(m + col, a.M - 1) * a.ldw;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    int k = 4 * grp;
    for (; k - 4 * grp + 64 <= a.K; k += 64) {                    // four steps' loads in flight together
        E fw[4][4], fx[4][4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            __builtin_memcpy(fw[u], w + k + 16 * u, 4 * sizeof(E));
            __builtin_memcpy(fx[u], x + k + 16 * u, 4 * sizeof(E));
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(load_f(&fw[u][i]), load_f(&fx[u][i]), acc, 0, 0, 0);
    }
    for (; k - 4 * grp < a.K; k += 16)
        for (int i = 0; i < 4; ++i) {
            const bool on = k + i < a.K;
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(on ? load_f(w + k + i) : 0.f, on ? load_f(x + k + i) : 0.f, acc, 0, 0, 0);
        }
    for (int r = 0; r < 4; ++r) {
        if (!odd[r]) continue;
        const int c = m + 4 * grp + r;
        float v = acc[r] + (a.bias ? load_f((const E*)a.bias + c) : 0.f);
        if (id >= 0) {
            float s = 0.f;
            for (int q = 0; q < a.r; ++q) s = fmaf(load_f((const E*)a.up + ((size_t)id * a.M + c) * a.r + q), z[q], s);
            v += s;
        }
        store_f(y + c, a.relu ? relu_(v) : v);
    }
}
template <class F, int... I>
static __device__ __forceinline__ void each_of(F& f, std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }
// where the piece (row % 16, group of eight elements 0..3) of a block lies
static __device__ __forceinline__ int block_piece(int row, int g) { return g * 16 + (row ^ (g & 1) * 2 ^ (g >> 1) * 12); }
template <class E, int WR, int WC, int MR, int MC, int BK, bool TWO, bool FUSED, bool DIRECT>
MP_KERNEL __launch_bounds__(64 * WR * WC, WR * WC >= 8 ? 2 : 1) void mp_adapt_gemm(AdaptArgs a, int rows, int ntr, int ntc) {
    using G = Gemm<E, WR, WC, MR, MC, BK, TWO, FUSED, DIRECT>;
    constexpr int P = G::P, KS = G::KS, UR = G::UR, RN = G::RN, NU = G::NU, TH = G::TH, RUN = P == 1 ? 8 : 4;
    extern __shared__ __align__(16) char gemm_lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, grp = lane >> 4;
    // workgroups are dealt to the 8 XCDs in turn: a run of tiles (columns fastest: one panel of x) to each, so that an XCD's L2
    // holds what its tiles share
    const int nt = ntr * ntc, per = (nt + 7) / 8, tile = (int)(blockIdx.x % 8) * per + (int)(blockIdx.x / 8);
    if (tile >= nt || (int)(blockIdx.x / 8) >= per) return;
    // rows [n0, n1) of the flattened (sequence, frame) list; FUSED: tiles of a sequence
    const int tps = FUSED ? (a.T + RN - 1) / RN : 1, seq = FUSED ? tile / tps : 0;
    const int n0 = FUSED ? seq * a.T + tile % tps * RN : tile / ntc * RN, n1 = FUSED ? (seq + 1) * a.T : rows;
    const int m0 = FUSED ? 0 : tile % ntc * G::CM, Mp = (a.M + 15) / 16 * 16;
    const int sid = FUSED ? a.ids[seq] : 0;
    const bool adapt = FUSED && sid >= 0 && sid < a.n;
    const E* src[NU];
    const int w64 = __builtin_amdgcn_readfirstlane(wave) * NU;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
        const int row = DIRECT ? (w64 + u) * 8 + lane / 8 : (tid + TH * u) / UR;
        const int kk = DIRECT ? (lane % 8 ^ (row >> 1 & 7)) * 8 : (tid + TH * u) % UR * RUN;
        if (row < RN) {
            const int n = min(n0 + row, n1 - 1), b = n / a.T;
            src[u] = (const E*)a.x + (size_t)b * a.sx[0] + (size_t)(n - b * a.T) * a.sx[1] + kk;
        } else {
            const int m = m0 + row - RN;
            src[u] = (const E*)a.w + (size_t)min(m, a.M - 1) * a.ldw + kk;
            if (FUSED && adapt && m >= Mp) src[u] = (const E*)a.down + ((size_t)sid * a.r + min(m - Mp, a.r - 1)) * a.K + kk;
        }
    }
    const int wr = wave % WR, wc = wave / WR;
    f32x4 acc[MC][MR] = {};
    Oct<E> oct[NU];
    int at[NU];
#pragma unroll
    for (int u = 0; u < NU; ++u) {
        const int row = (tid + TH * u) / UR, o = (tid + TH * u) % UR;
        at[u] = (row / 16 * KS + o / 4) * 1024 + block_piece(row % 16, o % 4) * 16;
    }
    const int mine = DIRECT ? col * 128 : block_piece(col, grp) * 16;
    auto piece = [&](const char* from, int p, int tile, int ks) {
        return *(const u32x4*)(DIRECT ? from + tile * 2048 + mine + (ks * 4 + grp ^ col >> 1) * 16 : from + p * G::kPlane + (tile * KS + ks) * 1024 + mine);
    };
    auto stage_from = [&](Oct<E> (&oct)[NU], char* to) {
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            u32x4 p[P];
            oct[u].planes(p);
#pragma unroll
            for (int i = 0; i < P; ++i) *(u32x4*)(to + i * G::kPlane + at[u]) = p[i];
        }
    };
    auto stage = [&](char* to) { stage_from(oct, to); };
    auto multiply = [&](const char* from) {
        if constexpr (DIRECT) {
            u32x4 fw[KS][MC][1], fx[KS][MR][1];
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
                for (int j = 0; j < MC; ++j) fw[ks][j][0] = piece(from, 0, RN / 16 + wc * MC + j, ks);
#pragma unroll
                for (int i = 0; i < MR; ++i) fx[ks][i][0] = piece(from, 0, wr * MR + i, ks);
            }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int i = 0; i < MR; ++i)
#pragma unroll
                    for (int j = 0; j < MC; ++j) acc[j][i] = mfma_planes(fw[ks][j], fx[ks][i], acc[j][i]);
            __builtin_amdgcn_sched_group_barrier(0x100, MC + 2, 0);
#pragma unroll
            for (int g = 0; g < KS * MR; ++g) {
                __builtin_amdgcn_sched_group_barrier(0x8, MC, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
            }
            return;
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            u32x4 fx[MR][P];
#pragma unroll
            for (int i = 0; i < MR; ++i)
#pragma unroll
                for (int p = 0; p < P; ++p) fx[i][p] = piece(from, p, wr * MR + i, ks);
#pragma unroll
            for (int j = 0; j < MC; ++j) {
                u32x4 fw[P];
#pragma unroll
                for (int p = 0; p < P; ++p) fw[p] = piece(from, p, RN / 16 + wc * MC + j, ks);
#pragma unroll
                for (int i = 0; i < MR; ++i) acc[j][i] = mfma_planes(fw, fx[i], acc[j][i]);
            }
        }
    };
    // whole tiles, each asking for the next one (the last for itself again: no branch around the loads, which would make them wait
    // for each other), then what is left of K -- small tiles, which are chains of latencies, ask for that beside the last product
    const int whole = a.K / BK;
    // small tiles ask for their rows' adapters beside the first tile of K: a latency less at the end
    constexpr bool kEarly = MR == 1;
    int id[MR];
    auto early = [&]() { id[0] = a.ids[min(n0 + wr * 16 + col, n1 - 1) / a.T]; };
    auto fetch_to = [&](Oct<E> (&oct)[NU], int t) {
#pragma unroll
        for (int u = 0; u < NU; ++u) oct[u].load_runs(src[u] + (size_t)t * BK, BK / 2);
    };
    auto fetch = [&](int t) { fetch_to(oct, t); };
    char* const other = gemm_lds + (TWO ? G::kOne : 0);
    if constexpr (DIRECT) {
        auto ask = [&](int t, char* to) {
#pragma unroll
            for (int u = 0; u < NU; ++u)
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src[u] + (size_t)t * BK),
                                                 (__attribute__((address_space(3))) void*)(to + (w64 + u) * 1024), 16, 0, 0);
        };
        ask(0, gemm_lds);
        __syncthreads();
        for (int t = 0; t < whole; ++t) {
            ask(min(t + 1, whole - 1), t & 1 ? gemm_lds : other);
            multiply(t & 1 ? other : gemm_lds);
            __syncthreads();
        }
    } else if constexpr (kEarly) {
        const int left = a.K - whole * BK;
        auto fetch_left = [&]() {
#pragma unroll
            for (int u = 0; u < NU; ++u) oct[u].load_some_runs(src[u] + (size_t)whole * BK, BK / 2, left - (tid + TH * u) % UR * RUN);
        };
        if (whole) fetch(0);
        else fetch_left();
        stage(gemm_lds);
        early();
        __syncthreads();
        for (int t = 0; t + 1 < whole; ++t) {
            fetch(t + 1);
            multiply(t & 1 ? other : gemm_lds);
            if (!TWO) __syncthreads();
            stage(t & 1 ? gemm_lds : other);
            __syncthreads();
        }
        const bool two = whole && left;                           // (a last tile behind the whole ones)
        if (two) fetch_left();
        multiply(whole && !(whole & 1) ? other : gemm_lds);
        __syncthreads();
        if (two) {
            stage(whole & 1 ? other : gemm_lds);
            __syncthreads();
            multiply(whole & 1 ? other : gemm_lds);
            __syncthreads();
        }
    } else {
        if constexpr (FUSED) {
            // one workgroup a CU, and a tile's products are shorter than its loads' way: two tiles are on theirs
            Oct<E> far[NU];
            if (whole) {
                fetch(0);
                __builtin_amdgcn_sched_barrier(0);                // (in this order: the loop waits for as many as are older)
                fetch_to(far, min(1, whole - 1));
                __builtin_amdgcn_sched_barrier(0);
                stage(gemm_lds);
                __syncthreads();
            }
            int t = 0;
            for (; t + 1 < whole; t += 2) {
                fetch(min(t + 2, whole - 1));
                multiply(gemm_lds);
                stage_from(far, other);
                __syncthreads();
                fetch_to(far, min(t + 3, whole - 1));
                multiply(other);
                stage(gemm_lds);
                __syncthreads();
            }
            if (t < whole) multiply(gemm_lds);
            __syncthreads();
        } else {
            if (whole) {
                fetch(0);
                stage(gemm_lds);
                __syncthreads();
            }
            for (int t = 0; t < whole; ++t) {
                fetch(min(t + 1, whole - 1));
                multiply(t & 1 ? other : gemm_lds);
                if (!TWO) __syncthreads();
                stage(t & 1 ? gemm_lds : other);
                __syncthreads();
            }
        }
        if (whole * BK < a.K) {
#pragma unroll
            for (int u = 0; u < NU; ++u)
                oct[u].load_some_runs(src[u] + (size_t)whole * BK, BK / 2, a.K - whole * BK - (tid + TH * u) % UR * RUN);
            stage(gemm_lds);                                      // (nobody reads either buffer here: a barrier ended the last round)
            __syncthreads();
            multiply(gemm_lds);
            __syncthreads();
        }
    }
    const int rlen = a.r;
    float* zl = (float*)gemm_lds;                                 // FUSED: [RN][kRowZ]
    if (FUSED && adapt) {
        const float sc = a.scale ? a.scale[sid] : 1.f;
        float bad = 0.f;                                          // stays 0 while everything is finite
#pragma unroll
        for (int j = 0; j < MC; ++j) {
            const int m = (wc * MC + j) * 16 - Mp + 4 * grp;
            if (m >= 0)
#pragma unroll
                for (int i = 0; i < MR; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (m + r < rlen) {
                            zl[((wr * MR + i) * 16 + col) * G::kRowZ + m + r] = sc * acc[j][i][r];
                            bad = fmaf(0.f, acc[j][i][r], bad);
                        }
        }
        if (P == 1) __syncthreads();
        else if (__syncthreads_or(bad != 0.f)) {
            for (int i = tid; i < RN * rlen; i += TH) {
                const int row = i / rlen, c = i % rlen;
                float* const z = zl + row * G::kRowZ + c;
                if (n0 + row < n1 && not_finite(*z)) *z = sc * plain_dot(row_of_x<E>(a, n0 + row), (const E*)a.down + ((size_t)sid * a.r + c) * a.K, a.K);
            }
            __syncthreads();
        }
    }
    // the adapters, for all rows of the wave at once where they share one
    bool same = true;
#pragma unroll
    for (int i = 0; i < MR; ++i) {
        if (!kEarly) id[i] = FUSED ? sid : a.ids[min(n0 + (wr * MR + i) * 16 + col, n1 - 1) / a.T];
        same = same && id[i] == __builtin_amdgcn_readfirstlane(id[0]);
    }
    const int id0 = __builtin_amdgcn_readfirstlane(id[0]);
    const bool wave_same = FUSED || __all(same);
    // z is fp32 whatever the inputs are: all three terms of it
    constexpr int PZ = 3;
    auto z_of = [&](int i) {
        return FUSED ? zl + ((wr * MR + i) * 16 + col) * G::kRowZ : a.ws + (size_t)min(n0 + (wr * MR + i) * 16 + col, n1 - 1) * rlen;
    };
    auto z_planes = [&](const float* z, int k, u32x4 (&pz)[PZ]) {
        Oct<float> oz;
        oz.load_some(z + k, rlen - k < 0 ? 0 : rlen - k);
        oz.planes(pz);
    };
    auto up_planes = [&](int ad, int j, int k, u32x4 (&pu)[P]) {
        const int m = m0 + (wc * MC + j) * 16 + col;
        Oct<E> ou;
        ou.load_some((const E*)a.up + ((size_t)ad * a.M + (m < a.M ? m : 0)) * rlen + k, rlen - k < 0 ? 0 : rlen - k);
        ou.planes(pu);
    };
    if (wave_same && id0 >= 0 && id0 < a.n)
        for (int r0 = 0; r0 < rlen; r0 += 32) {
            u32x4 pu[MC][P];
#pragma unroll
            for (int j = 0; j < MC; ++j) up_planes(id0, j, r0 + 8 * grp, pu[j]);
            auto add = [&](auto tile_row) {
                constexpr int i = decltype(tile_row)::value;
                u32x4 pz[PZ];
                z_planes(z_of(i), r0 + 8 * grp, pz);
#pragma unroll
                for (int j = 0; j < MC; ++j) acc[j][i] = mfma_planes(pu[j], pz, acc[j][i]);
            };
            each_of(add, std::make_integer_sequence<int, MR>{});
        }
    // the bias of the lane's columns
    float bias[MC][4];
#pragma unroll
    for (int j = 0; j < MC; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int m = m0 + (wc * MC + j) * 16 + 4 * grp + r;
            bias[j][r] = a.bias && m < a.M ? load_f((const E*)a.bias + m) : 0.f;
        }
    // one 16-row tile of the wave (a function of a constant: acc stays in registers whatever the compiler thinks of unrolling this)
    const bool flat = a.sy[0] == (long)a.T * a.sy[1];
    auto row_of = [&](int n) {
        const int b = flat ? 0 : n / a.T;
        return (E*)a.y + (size_t)b * a.sy[0] + (size_t)(n - b * a.T) * a.sy[1];
    };
    float odd = 0.f;                                              // stays 0 while every result is finite
    auto finish = [&](auto tile_row) {
        constexpr int i = decltype(tile_row)::value;
        const int nt0 = n0 + (wr * MR + i) * 16, n = nt0 + col;    // 16 rows, one per lane column
        if (!wave_same) {
            const float* z = z_of(i);
            const int tid0 = __builtin_amdgcn_readfirstlane(id[i]);
            if (__all(id[i] == tid0)) {
                if (tid0 >= 0 && tid0 < a.n)                      // one adapter for the 16 rows: the matrix units again
                    for (int r0 = 0; r0 < rlen; r0 += 32) {
                        u32x4 pz[PZ], pu[P];
                        z_planes(z, r0 + 8 * grp, pz);
#pragma unroll
                        for (int j = 0; j < MC; ++j) {
                            up_planes(tid0, j, r0 + 8 * grp, pu);
                            acc[j][i] = mfma_planes(pu, pz, acc[j][i]);
                        }
                    }
            } else if (id[i] >= 0 && id[i] < a.n) {               // a row of its own each: dot products of the lane's four columns
                for (int q = 0; q < rlen; q += 8) {
                    Oct<float> oz;
                    oz.load_some(z + q, rlen - q);
#pragma unroll
                    for (int j = 0; j < MC; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int m = m0 + (wc * MC + j) * 16 + 4 * grp + r;
                            Oct<E> ou;
                            ou.load_some((const E*)a.up + ((size_t)id[i] * a.M + (m < a.M ? m : 0)) * rlen + q, rlen - q);
                            acc[j][i][r] = ou.dot(oz, acc[j][i][r]);
                        }
                }
            }
        }
        auto value = [&](int j, float (&y)[4]) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                y[r] = acc[j][i][r] + bias[j][r];
                odd = fmaf(0.f, y[r], odd);
                if (id[i] >= a.n) y[r] = __builtin_nanf("");
                if (a.relu) y[r] = relu_(y[r]);
            }
        };
        if (G::kTurn && a.vec == 2) {
            // whole lines: the wave's 16 rows x 16 MC columns through its own piece of LDS (the operands' place: a barrier ended
            // their last reads), 16 bytes a lane, the pieces of a row exchanged by its index against bank conflicts
            constexpr int PR = MC * 16 * sizeof(E) / 16;          // 16-byte pieces of a row
            char* const own = gemm_lds + ((wave * MR + i) * 16) * PR * 16;
#pragma unroll
            for (int j = 0; j < MC; ++j) {
                float y[4];
                value(j, y);
                const int byte = (j * 16 + 4 * grp) * sizeof(E);
                store4((E*)(own + (col * PR + (byte / 16 ^ col % PR)) * 16 + byte % 16), y);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int q = 0; q < PR / 4; ++q) {
                const int row = (q * 64 + lane) / PR, piece = lane % PR, m = m0 + wc * MC * 16 + piece * 16 / (int)sizeof(E);
                const u32x4 v = *(const u32x4*)(own + (row * PR + (piece ^ row % PR)) * 16);
                if (nt0 + row < n1 && m < a.M) *(u32x4*)(row_of(nt0 + row) + m) = v;
            }
            return;
        }
        if (n >= n1) return;
        E* const yrow = row_of(n);
#pragma unroll
        for (int j = 0; j < MC; ++j) {
            const int m = m0 + (wc * MC + j) * 16 + 4 * grp;
            float y[4];
            value(j, y);
            if (a.vec) {                                          // M a multiple of 4: whole groups of columns, aligned
                if (m < a.M) store4(yrow + m, y);
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (m + r < a.M) store_f(yrow + m + r, y[r]);
            }
        }
    };
    each_of(finish, std::make_integer_sequence<int, MR>{});
    if (__any(odd != 0.f)) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "agent");        // (the outputs are looked at again)
#pragma unroll 1
        for (int t = 0; t < MR * MC; ++t) {
            const int n = n0 + (wr * MR + t % MR) * 16, m = m0 + (wc * MC + t / MR) * 16, row = min(n + col, n1 - 1);
            if (n < n1 && m < a.M) plain_tile<E>(a, n, n1, m, FUSED ? zl + (row - n0) * G::kRowZ : a.ws + (size_t)row * rlen);
        }
    }
}

template <class E, int WR, int WC, int MR, int MC, int BK, bool TWO, bool FUSED = false, bool DIRECT = false>
static bool gemm_for(const AdaptArgs& a, int rows, hipStream_t s) {
    using G = Gemm<E, WR, WC, MR, MC, BK, TWO, FUSED, DIRECT>;
    const auto kernel = mp_adapt_gemm<E, WR, WC, MR, MC, BK, TWO, FUSED, DIRECT>;
    // (an attribute of the function on the current device: set at every launch, a call may come from any device's handle)
    if (G::kBytes > 64 * 1024 && hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, G::kBytes) != hipSuccess) return false;
    const int ntr = FUSED ? a.B * ((a.T + G::RN - 1) / G::RN) : (rows + G::RN - 1) / G::RN, ntc = FUSED ? 1 : (a.M + G::CM - 1) / G::CM;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((ntr * ntc + 7) / 8 * 8)), dim3(G::TH), G::kBytes, s, a, rows, ntr, ntc);
    return true;
}
template <class E>
static bool launch_for(AdaptArgs a, hipStream_t s) {
    constexpr bool half = Arith<E>::P == 1;
    const int rows = a.B * a.T;
    auto whole = [&](int n) { return a.M % n == 0 && a.sy[0] % n == 0 && a.sy[1] % n == 0 && (uintptr_t)a.y % (n * sizeof(E)) == 0; };
    a.vec = whole(16 / sizeof(E)) ? 2 : whole(4) ? 1 : 0;
    bool ok;
    // One launch that reads x once (FUSED) or two.  Its row tiles of 128 end with their sequence, its one column of tiles walks K in a
    // chain.  With many rows it wins (us, one against two): 256 x 125 512 -> 96 bf16 15 / 32, fp32 31 / 49; 128 x 125 fp32 29 / 35;
    // below 12000 rows the chain is what is timed (fp32 64 x 125 27 / 26, 8 x 125 26 / 16), unless K is short enough that the second
    // launch costs more (bf16 256 x 1 13 / 16, at K = 2048 30 / 16; fp32 K = 132 14 / 16); more row tiles than CUs have to be more than
    // half full (fp32 256 x 64 30 / 33, 1024 x 64 109 / 86, bf16 1024 x 1 30 / 16).
    const long ftiles = (long)a.B * ((a.T + 127) / 128);
    const bool few = ftiles <= 256, many_rows = rows >= 12000 && (few || rows > 64 * ftiles);
    if ((a.M + 15) / 16 * 16 + a.r <= 128 && (many_rows || (few && a.K <= (half ? 512 : 192)))) {
        ok = gemm_for<E, 4, 2, 2, 4, half ? 64 : 32, true, true>(a, rows, s);
        return hipGetLastError() == hipSuccess && ok;
    }
    auto down = [&](auto groups) {
        constexpr int RG = decltype(groups)::value;
        const int per_seq = (a.T + 16 * RG - 1) / (16 * RG);
        const dim3 grid((unsigned)(a.B * per_seq));
        if (a.r <= 16) hipLaunchKernelGGL((mp_adapt_down<E, 1, RG>), grid, dim3(256), 0, s, a, per_seq);
        else if (a.r <= 32) hipLaunchKernelGGL((mp_adapt_down<E, 2, RG>), grid, dim3(256), 0, s, a, per_seq);
        else if (a.r <= 64) hipLaunchKernelGGL((mp_adapt_down<E, 4, 1>), dim3((unsigned)(a.B * ((a.T + 15) / 16))), dim3(256), 0, s, a, (a.T + 15) / 16);
        else hipLaunchKernelGGL((mp_adapt_down<E, 8, 1>), dim3((unsigned)(a.B * ((a.T + 15) / 16))), dim3(256), 0, s, a, (a.T + 15) / 16);
    };
    // long sequences that fill the chip with groups of 32 frames read Down half as often (8 x 2048, K 2048, r 32: 18 us against 25)
    if (a.T >= 64 && rows >= 8192) down(std::integral_constant<int, 2>{});
    else down(std::integral_constant<int, 1>{});
    // The largest tile that leaves enough of them for 256 CUs (us, K = 1024, larger / smaller tile).  256: bf16 6144 x 2048 (192 tiles)
    // 43 / 58, 4096 x 2048 (128) 41 / 36.  128: bf16 4096 x 2048 (512) 37 / 44, 4096 x 1024 (256) 32 / 28; fp32, whose products take
    // three times as long, 4096 x 1024 (256) 60 / 76, 2048 x 1024 (128) 57 / 47.  64: 1024 x 1024 (256) bf16 15.9 / 16.2, fp32 38 / 39,
    // 768 x 1024 (192) 16.0 / 15.7 and 38 / 29.
    auto tiles = [&](int t) { return ((long)rows + t - 1) / t * ((a.M + t - 1) / t); };
    if constexpr (half)
        if (tiles(256) >= 192) {
            // rows of whole cache lines go to LDS directly, others through registers (8 x 2048, 2048 -> 2048: 174 us against 192 before the
            // steps that both share)
            const bool lines = a.K % 64 == 0 && a.ldw % 8 == 0 && a.sx[0] % 8 == 0 && a.sx[1] % 8 == 0 && ((uintptr_t)a.x | (uintptr_t)a.w) % 16 == 0;
            ok = lines ? gemm_for<E, 2, 4, 8, 4, 64, true, false, true>(a, rows, s) : gemm_for<E, 2, 4, 8, 4, 64, true>(a, rows, s);
            return hipGetLastError() == hipSuccess && ok;
        }
    constexpr int wr128 = half ? 2 : 4, mr128 = half ? 4 : 2;
    if (tiles(128) >= (half ? 384 : 192)) ok = gemm_for<E, wr128, 2, mr128, 4, half ? 64 : 32, !half>(a, rows, s);
    else if (tiles(64) >= 256) ok = gemm_for<E, 2, 2, 2, 2, half ? 128 : 64, false>(a, rows, s);
    else ok = gemm_for<E, 2, 2, 1, 1, half ? 256 : 128, false>(a, rows, s);
    return hipGetLastError() == hipSuccess && ok;
}
bool launch_adapt(const AdaptArgs& a, int dtype, hipStream_t s) {
    return dtype == kBF16 ? launch_for<bf16raw>(a, s) : launch_for<float>(a, s);
}

}  // namespace mpseq
