// The gated delta rule: a recurrence with a matrix state S [dk][dv] per sequence and value head, over whole sequences in chunks
// (launch_delta) and one frame per stream and tick (launch_delta_online).  Per frame t
//   S <- e^{g_t} S;   u_t = beta_t (v_t - S^T k_t);   S <- S + k_t u_t^T;   o_t = scale S^T q_t.
//
// Over a chunk of C = 32 frames that starts from S0, with G_i = g_1 + .. + g_i and D_ij = e^{G_i - G_j}:
//   A_ij = beta_i D_ij (k_i . k_j)  for j < i,     (I + A) U = diag(beta) (V - diag(e^G) K S0),
//   O = scale (diag(e^G) Q S0 + (tril(Q K^T) o D) U),     S' = e^{G_C} S0 + (diag(e^{G_C - G}) K)^T U.
// All products are matrix products; what does not depend on S0 -- (I + A)^{-1} and tril(Q K^T) o D -- is computed for all chunks
// at once (mp_delta_prep), the walk over the chunks (mp_delta_scan) carries S in registers.
//
// The decays come from the prefix sum G in 64 bits, per pair as e^{G_i - G_j}: a frame with g = -1e4 (a reset of the state) would
// cost the frames behind it their low bits if G were a float, and e^{G_i} / e^{G_j} would be 0 / 0.  g below -1e4 counts as -1e4
// (e^-104 already is 0 in fp32).
//
// A value that is not finite (or too large for a first bf16 term, 3.396e38) reaches the frames behind it only, as in the recurrence: where a
// right-hand side holds one, the rows from there on are taken out of the products (0 * NaN in a triangular matrix's zeros would
// reach the frames before it) and their outputs and the column's state are NaN.
#include "mp_seq_dev.h"

namespace mpseq {

constexpr int kC = 32;                            // frames per chunk
// Workspace of one (sequence, value head, chunk), bytes: T = (I + A)^{-1} diag(beta) and P = scale tril(Q K^T) o D as three terms each, in
// the order in which a lane of v_mfma_f32_16x16x32_bf16 takes its A operand, behind e^G and e^{G_C - G} of the 32 frames.  (Three
// beside bf16 outputs as well: with two of P, of U beside it and of the S in Q S0 the outputs of 8 x 2048 frames were not the
// correctly rounded ones in 0.23 % instead of 0.01 % of all places, in 173 us instead of 188.)
constexpr int kFrag = 1024;                       // one 16 x 32 operand: 64 lanes x 8 bf16
constexpr int kWsEg = 0, kWsTail = 4 * kC, kWsT = 8 * kC, kWsP = kWsT + 6 * kFrag, kWsUnit = kWsP + 6 * kFrag;

// Which frame and which component of k a lane's registers stand for.  The accumulator layout of a 16 x 16 tile (lane: column
// lane % 16, rows 4 (lane / 16) + r) becomes the B operand of a K = 32 instruction (lane: column lane % 16, k slots
// 8 (lane / 16) + 0..7) by putting two tiles h = 0, 1 side by side: row 4 g + r of tile h is index 8 g + 4 h + r of 32.  So the
// state (32 components per pair of tiles), the right-hand sides and U (32 frames per pair) go from one product into the next
// without leaving their lanes; the A operands take their rows in the same order.
static __device__ __forceinline__ int row_index(int h, int row) { return 8 * (row >> 2) + 4 * h + (row & 3); }

static __device__ __forceinline__ int length_of(const int* lengths, int b, int T) {
    if (!lengths) return T;
    const int n = lengths[b];
    return n < 0 ? 0 : n > T ? T : n;
}
static __device__ __forceinline__ f32x4 mfma4(float4 a, float4 b, f32x4 c) {
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.x, b.x, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.y, b.y, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.z, b.z, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a.w, b.w, c, 0, 0, 0);
}
static __device__ __forceinline__ float clamp_g(float g) { return g < -1e4f ? -1e4f : g; }      // (NaN stays NaN)
static __device__ __forceinline__ bool not_finite(float x) { return !(fabsf(x) <= 3.402823466e38f); }

// Components d .. d + 7 of a row of q or k, without a branch around the load (a branch would make the loads wait for each other):
// the address is moved inside the row, fix() puts zeros where the row or the sequence has ended.  MODE 0: dk is a multiple of 8;
// 1: it is not, but at least 8 -- the last eight components are loaded and shifted down; 2: dk < 8 or dv < 8, value by value.
template <class E, int MODE>
static __device__ __forceinline__ void load_oct(Oct<E>& o, const E* row, int d, int dk) {
    if (MODE == 0) o.load(row + (d < dk ? d : 0));
    else if (MODE == 1) o.load(row + min(d, dk - 8));
    else o.load_clamped(row, d, dk);
}
template <class E, int MODE>
static __device__ __forceinline__ void fix_oct(Oct<E>& o, int d, int dk, bool on) {
    if (MODE == 1) o.shift(d - min(d, dk - 8));
    if (MODE == 2) o.keep(dk - d);
    if (!on || d >= dk) o.zero();
}

// e^x of a difference of 64-bit prefix sums: the product with log2(e) in 64 bits, one rounding, the hardware's 2^x (1 ulp)
static __device__ __forceinline__ float decay(double x) { return __builtin_amdgcn_exp2f((float)(x * 1.4426950408889634)); }
// x of the lane `n` below within 16 lanes (0 where there is none); CTRL 0x142: of the last lane of the 16 before, in every second 16
template <int CTRL>
static __device__ __forceinline__ double lane_below(double x) {
    const long long v = __builtin_bit_cast(long long, x);
    constexpr int rows = CTRL == 0x142 ? 0xa : 0xf;
    const int lo = __builtin_amdgcn_update_dpp(0, (int)v, CTRL, rows, 0xf, true), hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, rows, 0xf, true);
    return __builtin_bit_cast(double, (long long)(unsigned)lo | (long long)hi << 32);
}

// One wave per (sequence, key head, chunk): K K^T and Q K^T once, then the value heads that share the key head.
// (I + A)^{-1} by forward substitution on the two 16 x 16 diagonal blocks -- a lane of two groups of 16 solves a column; stable
// where keys repeat and A is far from small, products of powers of A are not -- and T21 = -T22 A21 T11 on the fp32 matrix
// instructions.  KB: steps of 32 components whose loads are in flight together.  Bound by memory, its own output being the larger part:
// 8 x 2048 frames, 8 / 16 heads of 128, bf16 36 us (149 MB, 4.1 TB/s), 256 x 125 frames, 4 heads of 64, fp32 22 us.
template <class E, int MODE, int KB>
MP_KERNEL __launch_bounds__(64) void mp_delta_prep(DeltaArgs a) {
    constexpr int P = Arith<E>::P, LS = kC + 4;
    __shared__ __align__(16) float At[kC][LS], Tm[kC][LS], betas[kC];      // A transposed: [column][row]
    __shared__ __align__(16) double Gs[kC];
    float (*W)[LS] = Tm;                          // P on its way into operand order, before T is there
    const int unit = blockIdx.x, c = unit % a.nchunk, hk = unit / a.nchunk % a.Hk, b = unit / a.nchunk / a.Hk;
    const int lane = threadIdx.x, col = lane & 15, grp = lane >> 4, i = lane & 31, t0 = c * kC;
    const int rep = a.Hv / a.Hk, t = t0 + i;
    const E* q = (const E*)a.q + b * a.sq[0] + hk * a.sq[2];
    const E* k = (const E*)a.k + b * a.sk[0] + hk * a.sk[2];
    const int len = length_of(a.lengths, b, a.T);
    if (t0 >= len) return;
    // (everything is requested at once; rows behind the sequence's end are not there: its last one instead, and dropped)
    const int tl[2] = {min(t0 + col, len - 1), min(t0 + 16 + col, len - 1)};
    Oct<E> ok[KB][2], oq[KB][2];
    auto request = [&](int d0) {
#pragma unroll
        for (int m = 0; m < KB; ++m)
#pragma unroll
            for (int I = 0; I < 2; ++I) {
                load_oct<E, MODE>(ok[m][I], k + tl[I] * a.sk[1], d0 + 32 * m + 8 * grp, a.dk);
                load_oct<E, MODE>(oq[m][I], q + tl[I] * a.sq[1], d0 + 32 * m + 8 * grp, a.dk);
            }
    };
    request(0);
    auto gate = [&](const float* p, const long (&s)[3], int e) { return p[b * s[0] + min(t, len - 1) * s[1] + (hk * rep + e) * s[2]]; };
    float gnext = gate(a.g, a.sg, 0), bnext = gate(a.beta, a.sb, 0);
    const bool on = t < len;
    f32x4 kk[3] = {}, qk[3] = {};                 // tiles (0,0), (1,0), (1,1) of frames 16 I + row, 16 J + column
    for (int d0 = 0; d0 < a.dk; d0 += 32 * KB) {
        if (d0) request(d0);
#pragma unroll
        for (int m = 0; m < KB; ++m) {
            u32x4 fk[2][P], fq[2][P];
            const int d = d0 + 32 * m + 8 * grp;
#pragma unroll
            for (int I = 0; I < 2; ++I) {
                fix_oct<E, MODE>(ok[m][I], d, a.dk, t0 + 16 * I + col < len);
                fix_oct<E, MODE>(oq[m][I], d, a.dk, t0 + 16 * I + col < len);
                ok[m][I].planes(fk[I]);
                oq[m][I].planes(fq[I]);
            }
#pragma unroll
            for (int n = 0; n < 3; ++n) {
                kk[n] = mfma_planes(fk[n > 0], fk[n > 1], kk[n]);
                qk[n] = mfma_planes(fq[n > 0], fk[n > 1], qk[n]);
            }
        }
    }
    char* ws = (char*)a.ws + ((size_t)(b * a.Hv + hk * rep) * a.nchunk + c) * kWsUnit;
    for (int e = 0; e < rep; ++e, ws += (size_t)a.nchunk * kWsUnit) {
        const float beta = on ? bnext : 0.f;
        double G = on ? (double)clamp_g(gnext) : 0.0;             // lanes 32.. as lanes 0..31
        if (e + 1 < rep) { gnext = gate(a.g, a.sg, e + 1); bnext = gate(a.beta, a.sb, e + 1); }
        G += lane_below<0x111>(G);
        G += lane_below<0x112>(G);
        G += lane_below<0x114>(G);
        G += lane_below<0x118>(G);
        G += lane_below<0x142>(G);
        const long long top = __builtin_bit_cast(long long, G);
        const double last = __builtin_bit_cast(double, (long long)(unsigned)__builtin_amdgcn_readlane((int)top, 31) |
                                                       (long long)__builtin_amdgcn_readlane((int)(top >> 32), 31) << 32);
        __syncthreads();
        if (lane < kC) {
            Gs[i] = G;
            betas[i] = beta;
            ((float*)(ws + kWsEg))[i] = decay(G);
            ((float*)(ws + kWsTail))[i] = decay(last - G);
        }
        __syncthreads();
        double Gr[2][4];
        float br[2][4];
#pragma unroll
        for (int I = 0; I < 2; ++I) {
            __builtin_memcpy(Gr[I], __builtin_assume_aligned(&Gs[16 * I + 4 * grp], 16), 32);
            __builtin_memcpy(br[I], __builtin_assume_aligned(&betas[16 * I + 4 * grp], 16), 16);
        }
        const double Gc[2] = {Gs[col], Gs[16 + col]};
#pragma unroll
        for (int tile = 0; tile < 3; ++tile) {
            const int I = tile > 0, J = tile > 1, cj = 16 * J + col;
            float av[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int ri = 16 * I + 4 * grp + r;
                const float D = decay(Gr[I][r] - Gc[J]);
                av[r] = cj < ri ? br[I][r] * D * kk[tile][r] : 0.f;
                W[ri][cj] = cj <= ri ? a.scale * D * qk[tile][r] : 0.f;
            }
            *(float4*)&At[cj][16 * I + 4 * grp] = {av[0], av[1], av[2], av[3]};
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) W[4 * grp + r][16 + col] = 0.f;
        __syncthreads();
#pragma unroll
        for (int I = 0; I < 2; ++I) {
            Oct<float> o;
            u32x4 p[3];
            o.load(&W[row_index(I, col)][8 * grp]);
            o.planes(p);
#pragma unroll
            for (int n = 0; n < 3; ++n) *(u32x4*)(ws + kWsP + (I * 3 + n) * kFrag + lane * 16) = p[n];
        }
        // the diagonal blocks (groups 2 and 3 as 0 and 1)
        const int blk = grp & 1;
        float x[16];
#pragma unroll
        for (int n = 0; n < 16; ++n) x[n] = n == col ? 1.f : 0.f;
#pragma unroll
        for (int n = 0; n < 15; ++n) {
            float an[16];
#pragma unroll
            for (int m = (n + 1) / 4; m < 4; ++m) __builtin_memcpy(&an[4 * m], __builtin_assume_aligned(&At[16 * blk + n][16 * blk + 4 * m], 16), 16);
            if (n < col) x[n] = 0.f;              // (not 0 * NaN where an earlier frame's row is not finite)
#pragma unroll
            for (int j = n + 1; j < 16; ++j) x[j] = fmaf(-an[j], x[n], x[j]);
        }
        if (15 < col) x[15] = 0.f;
        __syncthreads();
#pragma unroll
        for (int n = 0; n < 16; ++n) {
            Tm[16 * blk + n][16 * blk + col] = x[n];
            if (blk == 0) Tm[n][16 + col] = 0.f;
        }
        __syncthreads();
        {
            f32x4 X = {0.f, 0.f, 0.f, 0.f}, T21 = {0.f, 0.f, 0.f, 0.f};
            const int l = 4 * grp;
            const float4 a21 = {At[l][16 + col], At[l + 1][16 + col], At[l + 2][16 + col], At[l + 3][16 + col]};
            const float4 t11 = {Tm[l][col], Tm[l + 1][col], Tm[l + 2][col], Tm[l + 3][col]};
            const float4 t22 = *(const float4*)&Tm[16 + col][16 + l];
            X = mfma4(a21, t11, X);
            float4 y;                                             // (a later frame's row that is not finite is kept from the zeros of T22,
                                                                  //  and is NaN itself: what hides in it may come from finite inputs)
            y.x = not_finite(X[0]) ? 0.f : X[0];
            y.y = not_finite(X[1]) ? 0.f : X[1];
            y.z = not_finite(X[2]) ? 0.f : X[2];
            y.w = not_finite(X[3]) ? 0.f : X[3];
            T21 = mfma4(t22, y, T21);
#pragma unroll
            for (int r = 0; r < 4; ++r) Tm[16 + l + r][col] = not_finite(X[r]) ? __builtin_nanf("") : -T21[r];
        }
        __syncthreads();
        float bc[8];
        __builtin_memcpy(bc, __builtin_assume_aligned(&betas[8 * grp], 16), 32);
#pragma unroll
        for (int I = 0; I < 2; ++I) {
            Oct<float> o;
            u32x4 p[3];
            const int row = row_index(I, col);
            o.load(&Tm[row][8 * grp]);
#pragma unroll
            for (int j = 0; j < 8; ++j) o.v[j] = 8 * grp + j > row ? 0.f : o.v[j] * bc[j];
            o.planes(p);
#pragma unroll
            for (int n = 0; n < 3; ++n) *(u32x4*)(ws + kWsT + (I * 3 + n) * kFrag + lane * 16) = p[n];
        }
    }
}

// The walk over the chunks: a workgroup per (sequence, value head, 64 columns of the state), a wave per 16 columns; NK = dk / 32
// rounded up.  The workgroup stages a chunk in LDS -- K and Q as ready operands (bf16 terms, one 16-byte read per lane and operand;
// K^T comes from K's operands by the turning reads), the chunk's workspace, the 64 columns of V, whose place the outputs take --
// and the next chunk is on its way through registers meanwhile, with no use of its values before this chunk's products are done.
// Bound by the chain of a chunk -- products with S, U, products with U, the new S split into terms again -- whose steps overlap between
// waves only: 8 x 2048 frames, 16 heads of 128, bf16 165 us, 2.6 us a chunk, the matrix units busy 20 % of it; 256 x 125, 4 heads of 64,
// fp32 48 us (17 %).  Two waves per 16 columns (each half of dk) took as long: what they share goes through LDS once more.
constexpr int kFragK = kFrag + 256;               // K's operands: 64 bytes between the groups of eight components, or the 16 lanes of a
                                                  // turning read would meet in a quarter of the banks
template <class E, int NK>
struct ScanLds {
    static constexpr int P = Arith<E>::P, kPlaneK = 2 * NK * kFragK, kPlaneQ = 2 * NK * kFrag;
    static constexpr int kQ = P * kPlaneK, kWs = kQ + P * kPlaneQ, kV = kWs + (kWsUnit + 15) / 16 * 16, kRowV = (64 + 16 / sizeof(E)) * sizeof(E);
    static constexpr int kBytes = kV + kC * kRowV;
};
template <class E, int NK, int MODE>
struct Rows {                                     // what a thread stages of a chunk
    using L = ScanLds<E, NK>;
    static constexpr int P = L::P, NF = (2 * NK + 3) / 4, kUnit = kWsUnit, NW = (kUnit + 4095) / 4096;
    Oct<E> k[NF], q[NF], v;
    u32x4 ws[NW];
    unsigned ok[NF], oq[NF], ov;                  // byte offsets from the chunk's first row
    static __device__ __forceinline__ int frame(int f) { return row_index(f & 1, threadIdx.x & 15); }
    static __device__ __forceinline__ int component(int f) { return 32 * (f >> 1) + 8 * (threadIdx.x >> 4 & 3); }
    __device__ __forceinline__ void place(const DeltaArgs& a, int last_row, int c0) {
        const int wave = threadIdx.x >> 6;
#pragma unroll
        for (int n = 0; n < NF; ++n) {
            const int f = min(wave + 4 * n, 2 * NK - 1), t = min(frame(f), last_row), d = component(f);
            const int at = MODE == 0 ? (d < a.dk ? d : 0) : MODE == 1 ? min(d, a.dk - 8) : 0;
            ok[n] = (unsigned)(t * (int)a.sk[1] + at) * sizeof(E);
            oq[n] = (unsigned)(t * (int)a.sq[1] + at) * sizeof(E);
        }
        const int col = c0 + 8 * (threadIdx.x & 7);
        ov = (unsigned)(min((int)threadIdx.x >> 3, last_row) * (int)a.sv[1] + (MODE == 2 ? 0 : min(col, a.dv - 8))) * sizeof(E);
    }
    __device__ __forceinline__ void load(const DeltaArgs& a, const char* kb, const char* qb, const char* vb, const char* wp, int c0) {
        const int tid = threadIdx.x, wave = tid >> 6;
#pragma unroll
        for (int n = 0; n < NW; ++n) ws[n] = *(const u32x4*)(wp + (unsigned)min(4096 * n + 16 * tid, kUnit - 16));
        if (MODE == 2) v.load_clamped((const E*)(vb + ov), c0 + 8 * (tid & 7), a.dv);
        else v.load((const E*)(vb + ov));
#pragma unroll
        for (int n = 0; n < NF; ++n) {
            if (MODE == 2) {
                const int d = component(min(wave + 4 * n, 2 * NK - 1));
                k[n].load_clamped((const E*)(kb + ok[n]), d, a.dk);
                q[n].load_clamped((const E*)(qb + oq[n]), d, a.dk);
            } else {
                k[n].load((const E*)(kb + ok[n]));
                q[n].load((const E*)(qb + oq[n]));
            }
        }
    }
    __device__ __forceinline__ void store(const DeltaArgs& a, char* lds, int t0, int len, int c0) {
        const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
        const bool edge = t0 + kC > len || a.dk != 32 * NK;       // (uniform) something of the 32 x 32 NK block is not there
#pragma unroll
        for (int n = 0; n < NW; ++n)
            if (4096 * n + 16 * tid < kUnit) *(u32x4*)(lds + L::kWs + 4096 * n + 16 * tid) = ws[n];
        const int col = c0 + 8 * (tid & 7);
        if (MODE != 2 && a.dv % 8) v.shift(col - min(col, a.dv - 8));
        if (t0 + (tid >> 3) >= len) v.zero();
        __builtin_memcpy(__builtin_assume_aligned(lds + L::kV + (tid >> 3) * L::kRowV + 8 * (tid & 7) * sizeof(E), 16), &v.v, sizeof(v.v));
#pragma unroll
        for (int n = 0; n < NF; ++n) {
            const int f = wave + 4 * n;
            if (f < 2 * NK) {
                u32x4 pk[P], pq[P];
                if (MODE != 0 || edge) {
                    fix_oct<E, MODE>(k[n], component(f), a.dk, t0 + frame(f) < len);
                    fix_oct<E, MODE>(q[n], component(f), a.dk, t0 + frame(f) < len);
                }
                k[n].planes(pk);
                q[n].planes(pq);
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    *(u32x4*)(lds + p * L::kPlaneK + f * kFragK + lane * 16 + (lane >> 4) * 64) = pk[p];
                    *(u32x4*)(lds + L::kQ + p * L::kPlaneQ + f * kFrag + lane * 16) = pq[p];
                }
            }
        }
        // what a branch above left unused: its registers would have to be waited for at the loop's top, behind the stores of the outputs
#pragma unroll
        for (int n = 0; n < NW; ++n) asm volatile("" ::"v"(ws[n]));
        v.arrived();
#pragma unroll
        for (int n = 0; n < NF; ++n) { k[n].arrived(); q[n].arrived(); }
    }
};
// Left to itself the compiler puts every LDS read in front of its use, and a lone wave waits for each.  (fp32: the operands of a
// step ahead are 96 registers more than a wave has beside another)
#define FENCE() do { if (P == 1) __builtin_amdgcn_sched_barrier(0); } while (0)
static __device__ __forceinline__ u32x4 operand(const char* p, int lane) { return *(const u32x4*)(p + lane * 16); }

// Few sequences and heads: the chunks are cut into segments that run side by side.  A segment maps the state it starts from linearly,
// S -> M S + N; N [dk][dv] is its run from zero, column j of M [dk][dk] its run from the j-th unit vector with V = 0: the same
// kernel without its outputs (OUT = false), dv + dk columns.  mp_delta_join carries the states through the segments, then all
// segments run from their own start (OUT = true).  Three times the work, in 2 / segments of the steps.  state_in may be state_out,
// and in the last pass the segment with a sequence's end writes that buffer while nothing orders it behind the first one: the first
// pass puts the start of every sequence aside for it, by the workgroups whose part of M would be the first segment's (by those that
// run it: 1 x 3000 frames 54.5 -> 58.5 us).
struct DeltaPlan {
    int nseg, len;                                // segments and chunks per segment; nseg = 1: the chunks in one go
    float *N, *M;                                 // [B][Hv][nseg - 1][dk][dv] (mp_delta_join turns N of s into the start of s + 1), [..][dk][dk]
    float* S0;                                    // [B][Hv][dk][dv]: the start of sequences that go on behind the first segment
};
template <class E, int NK> constexpr bool two_per_cu() { return Arith<E>::P == 1 ? NK <= 4 : NK <= 2; }
template <class E, int NK, int MODE, bool OUT>
MP_KERNEL __launch_bounds__(256, (two_per_cu<E, NK>() ? 2 : 1)) void mp_delta_scan(DeltaArgs a, DeltaPlan plan, int ncol, int ncolm) {
    using L = ScanLds<E, NK>;
    constexpr int P = L::P;
    extern __shared__ __align__(16) char scan_lds[];
    char* const lds = scan_lds;
    const char* const ws = lds + L::kWs;
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, grp = lane >> 4;
    // the workgroups that read the same K and Q on one XCD (workgroups are dealt to the 8 of them in turn)
    const int rep = a.Hv / a.Hk, nc_all = ncol + ncolm, inner = rep * nc_all, nseg = OUT ? plan.nseg : plan.nseg - 1;
    const int rest = blockIdx.x >> 3, unit = rest / inner * 8 + (blockIdx.x & 7);
    if (unit >= a.B * a.Hk * nseg) return;
    const int seg = unit / (a.B * a.Hk), hk = unit % a.Hk, b = unit / a.Hk % a.B, hv = hk * rep + rest % inner / nc_all;
    const bool unitcol = !OUT && rest % nc_all >= ncol;            // columns of M
    const int c0 = 64 * (unitcol ? rest % nc_all - ncol : rest % nc_all), cv = c0 + 16 * (tid >> 6) + col;
    const int width = unitcol ? a.dk : a.dv;
    const bool cok = cv < width;
    const int len_all = length_of(a.lengths, b, a.T);
    // this segment's frames, as a sequence that begins at its first
    const int s0 = seg * plan.len * kC, len = min(len_all, seg + 1 == plan.nseg ? a.T : s0 + plan.len * kC) - s0;
    if (!OUT && len_all <= s0 + plan.len * kC) return;             // (no segment follows)
    if (!OUT && unitcol && seg == 0) {                             // (the first one's start is known: nothing to run, but put it aside)
        const size_t at = (size_t)(b * a.Hv + hv) * a.dk * a.dv;
        if (a.s_in)
            for (int i = c0 * a.dv + tid; i < min(c0 + 64, a.dk) * a.dv; i += 256) plan.S0[at + i] = a.s_in[at + i];
        return;
    }
    const char* q = (const char*)((const E*)a.q + b * a.sq[0] + hk * a.sq[2] + s0 * a.sq[1]);
    const char* k = (const char*)((const E*)a.k + b * a.sk[0] + hk * a.sk[2] + s0 * a.sk[1]);
    const char* v = (const char*)((const E*)a.v + b * a.sv[0] + hv * a.sv[2] + s0 * a.sv[1]);
    const long kstep = kC * a.sk[1] * sizeof(E), qstep = kC * a.sq[1] * sizeof(E), vstep = kC * a.sv[1] * sizeof(E);
    const char* wsg = (const char*)a.ws + ((size_t)(b * a.Hv + hv) * a.nchunk + seg * plan.len) * kWsUnit;
    const size_t so = (size_t)a.Hv * a.dv, head = (size_t)(b * a.Hv + hv), cc = cok ? cv : width - 1;
    const float* s_in = seg == 0 ? a.s_in : OUT ? plan.N + (head * (plan.nseg - 1) + seg - 1) * a.dk * a.dv : nullptr;
    if (seg == 0 && s_in) s_in = (OUT && len_all > plan.len * kC ? plan.S0 : s_in) + head * a.dk * a.dv;
    const int tmax = a.T - s0;                                     // frames of the tensor from here on
    // outputs leave as eight columns of a frame per thread, from the place of V
    const int ocol = c0 + 8 * (tid & 7), ofull = a.dv - ocol;
    E* o = (E*)a.o + (((size_t)b * a.T + s0) * a.Hv + hv) * a.dv + (size_t)(tid >> 3) * so + ocol;
    char* const oplace = lds + L::kV + (tid >> 3) * L::kRowV + 8 * (tid & 7) * sizeof(E);
    char* const vplace = lds + L::kV + 8 * grp * L::kRowV + (16 * (tid >> 6) + col) * sizeof(E);
    const int turned = (4 * grp + (col >> 2)) * 16 + (col & 3) * 320;      // this lane's piece of a turning read of K's operands
    f32x4 S[2 * NK];
#pragma unroll
    for (int n = 0; n < 2 * NK; ++n) S[n] = (f32x4){0.f, 0.f, 0.f, 0.f};
    if (unitcol) {
#pragma unroll
        for (int n = 0; n < 2 * NK; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) S[n][r] = 32 * (n >> 1) + row_index(n & 1, 4 * grp + r) == cv ? 1.f : 0.f;
    } else if (s_in) {
#pragma unroll
        for (int n = 0; n < 2 * NK; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int d = 32 * (n >> 1) + row_index(n & 1, 4 * grp + r);
                const float x = s_in[cc + (size_t)min(d, a.dk - 1) * a.dv];
                S[n][r] = d < a.dk ? x : 0.f;
            }
    }
    const float nan = __builtin_nanf("");
    const int nc = len <= 0 ? 0 : (len + kC - 1) / kC;
    Rows<E, NK, MODE> rows;
    if (nc > 0) {
        rows.place(a, min(kC, len) - 1, c0);
        rows.load(a, k, q, v, wsg, c0);
        rows.store(a, lds, 0, len, c0);
    }
    __syncthreads();
    for (int c = 0; c < nc; ++c) {
        const int t0 = c * kC;
        if (c + 1 < nc) {                                          // (the last chunk asks for itself again: no branch around the loads)
            k += kstep; q += qstep; v += vstep; wsg += kWsUnit;
            if (t0 + 2 * kC > len) rows.place(a, len - 1 - t0 - kC, c0);     // (rows behind the sequence's end are not there)
        }
        rows.load(a, k, q, v, wsg, c0);
        __builtin_amdgcn_sched_barrier(0);                         // (the loads are issued here, not where their values are used)
        // (requested in front of the products that they wait for)
        FENCE();
        float eg[8], tail[8];
        __builtin_memcpy(eg, __builtin_assume_aligned(ws + kWsEg + 32 * grp, 16), 32);
        u32x4 T[2][3];
#pragma unroll
        for (int I = 0; I < 2; ++I)
#pragma unroll
            for (int p = 0; p < 3; ++p) T[I][p] = operand(ws + kWsT + (I * 3 + p) * kFrag, lane);
        E vv[8];
        if (P == 1) {
            const char* at = lds + L::kV + (8 * grp + (col >> 2)) * L::kRowV + (16 * (tid >> 6) + 4 * (col & 3)) * sizeof(E);
            const uint2 x[2] = {read_turned(at), read_turned(at + 4 * L::kRowV)};
            __builtin_memcpy(vv, x, 16);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) vv[j] = *(const E*)(vplace + j * L::kRowV);
        }
        // K S0 and Q S0, one pair of state tiles (32 components) a step: the operands and the terms of the next step are made while
        // this one is multiplied
        f32x4 kq[4] = {};                                          // K S0: 0, 1, Q S0: 2, 3
        u32x4 f[2][4][P], sp[2][3];
        auto request = [&](int m) {
#pragma unroll
            for (int I = 0; I < 2; ++I)
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    f[m & 1][I][p] = *(const u32x4*)(lds + p * L::kPlaneK + (2 * m + I) * kFragK + lane * 16 + grp * 64);
                    if (OUT) f[m & 1][2 + I][p] = operand(lds + L::kQ + p * L::kPlaneQ + (2 * m + I) * kFrag, lane);
                }
        };
        auto split = [&](int m) {
            Oct<float> os;
#pragma unroll
            for (int j = 0; j < 8; ++j) os.v[j] = S[2 * m + (j >> 2)][j & 3];
            os.planes(sp[m & 1]);
        };
        request(0);
        split(0);
#pragma unroll
        for (int m = 0; m < NK; ++m) {
            FENCE();
            if (m + 1 < NK) request(m + 1);
            FENCE();
            if (!OUT) {
                u32x4 fk[2][P];
                f32x4 k2[2] = {kq[0], kq[1]};
#pragma unroll
                for (int p = 0; p < P; ++p) { fk[0][p] = f[m & 1][0][p]; fk[1][p] = f[m & 1][1][p]; }
                mfma_planes_n<2, P, 3>(fk, sp[m & 1], k2);
                kq[0] = k2[0];
                kq[1] = k2[1];
            } else {
                mfma_planes_n<4, P, 3>(f[m & 1], sp[m & 1], kq);
            }
            if (m + 1 < NK) {
                split(m + 1);
#pragma unroll
                for (int i = 0; i < (OUT ? P == 1 ? 12 : 24 : P == 1 ? 6 : 12); ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);                 // a matrix instruction,
                    __builtin_amdgcn_sched_group_barrier(0x2, P == 1 ? 5 : 2, 0);    // vector instructions that fit behind it
                }
            }
        }
        FENCE();
        __builtin_memcpy(tail, __builtin_assume_aligned(ws + kWsTail + 32 * grp, 16), 32);
        const float whole = *(const float*)(ws + kWsEg + 4 * (kC - 1));
        Oct<float> R;
        float odd = 0.f;                                           // stays 0 while everything is finite
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            R.v[j] = fmaf(-eg[j], kq[j >> 2][j & 3], unitcol ? 0.f : load_f(&vv[j]));
            odd = fmaf(0.f, R.v[j], odd);
        }
        bool any_bad = __any(cok && odd != 0.f);
        int first = kC;                                            // this column's first row that is not finite
        auto find_first = [&](const Oct<float>& x) {
#pragma unroll
            for (int j = 7; j >= 0; --j)
                if (not_finite(x.v[j])) first = min(first, 8 * grp + j);
            first = min(first, __shfl_xor(first, 16));
            first = min(first, __shfl_xor(first, 32));
        };
        if (any_bad) {
            find_first(R);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (8 * grp + j >= first) R.v[j] = 0.f;
        }
        u32x4 rp[3];
        R.planes(rp);
        u32x4 Pm[2][3], ft[2][4][P];
        auto turn = [&](int m) {
#pragma unroll
            for (int n = 0; n < 4 && 4 * m + n < 2 * NK; ++n)
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    const char* at = lds + p * L::kPlaneK + ((4 * m + n) & ~1) * kFragK + turned + 8 * (n & 1);
                    const uint2 lo = read_turned(at), hi = read_turned(at + kFragK);
                    ft[m & 1][n][p] = (u32x4){lo.x, lo.y, hi.x, hi.y};
                }
        };
        FENCE();
        turn(0);
#pragma unroll
        for (int I = 0; I < 2; ++I)
#pragma unroll
            for (int p = 0; p < 3; ++p)
                if (OUT) Pm[I][p] = operand(ws + kWsP + (I * 3 + p) * kFrag, lane);
        FENCE();
        f32x4 u[2] = {}, w[2] = {};
        mfma_planes_n<2, 3, 3>(T, rp, u);
        Oct<float> U, Ut;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            U.v[j] = u[j >> 2][j & 3];
            odd = fmaf(0.f, U.v[j], odd);
        }
        if (__any(cok && odd != 0.f)) {                            // (beta is in T)
            any_bad = true;
            find_first(U);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (8 * grp + j >= first) U.v[j] = 0.f;
        }
        // S' = e^{G_C} S0 + K^T (e^{G_C - G} U), four tiles a step, and P U beside it
#pragma unroll
        for (int j = 0; j < 8; ++j) Ut.v[j] = tail[j] * U.v[j];
        u32x4 up[3], ut[3];
        Ut.planes(ut);
        if (OUT) U.planes(up);
#pragma unroll
        for (int m = 0; m < (NK + 1) / 2; ++m) {
            FENCE();
            if (4 * m + 4 < 2 * NK) turn(m + 1);
            FENCE();
            if (4 * m + 4 <= 2 * NK) {
                f32x4 s4[4];
#pragma unroll
                for (int n = 0; n < 4; ++n) s4[n] = S[4 * m + n] * whole;
                mfma_planes_n<4, P, 3>(ft[m & 1], ut, s4);
#pragma unroll
                for (int n = 0; n < 4; ++n) S[4 * m + n] = s4[n];
            } else {
#pragma unroll
                for (int n = 0; n < 2; ++n) S[4 * m + n] = mfma_planes(ft[m & 1][n], ut, S[4 * m + n] * whole);
            }
        }
        if (OUT) mfma_planes_n<2, 3, 3>(Pm, up, w);
#pragma unroll
        for (int j = 0; OUT && j < 8; ++j) {
            float ov = fmaf(a.scale * eg[j], kq[2 + (j >> 2)][j & 3], w[j >> 2][j & 3]);
            if (any_bad && 8 * grp + j >= first) ov = nan;
            store_f((E*)(vplace + j * L::kRowV), ov);
        }
        if (any_bad && first < kC)
#pragma unroll
            for (int n = 0; n < 2 * NK; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r) S[n][r] = nan;
        __syncthreads();
        Oct<E> out;
        if (OUT) __builtin_memcpy(&out.v, __builtin_assume_aligned(oplace, 16), sizeof(out.v));
        // (the last chunk as well, its own rows again: loads that may stay unused would have to be waited for at the loop's top, behind
        //  the stores of the outputs)
        rows.store(a, lds, t0 + kC, len, c0);
        __syncthreads();
        if (OUT && t0 + (tid >> 3) < len) {
            E* at = o + (size_t)t0 * so;
            if (ofull >= 8) __builtin_memcpy(at, &out.v, sizeof(out.v));
            else {
                E e[8];
                __builtin_memcpy(e, &out.v, sizeof(e));
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < ofull) at[i] = e[i];
            }
        }
    }
    float* s_out = nullptr;
    size_t pitch = a.dv;
    if (OUT) {
        const int end = seg + 1 == plan.nseg ? tmax : min(tmax, plan.len * kC);
        for (int t = max(len, 0) + (tid >> 3); t < end; t += 32) {
            E* at = o + (size_t)(t - (tid >> 3)) * so;
            for (int i = 0; i < min(8, ofull); ++i) at[i] = 0;
        }
        // the segment with the sequence's last frame
        if (a.s_out && (len > 0 || seg == 0) && (seg + 1 == plan.nseg || len_all <= s0 + plan.len * kC)) s_out = a.s_out + head * a.dk * a.dv;
    } else {
        pitch = width;
        s_out = unitcol ? plan.M + (head * (plan.nseg - 1) + seg) * a.dk * a.dk : plan.N + (head * (plan.nseg - 1) + seg) * a.dk * a.dv;
    }
    if (s_out && cok)
#pragma unroll
        for (int n = 0; n < 2 * NK; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int d = 32 * (n >> 1) + row_index(n & 1, 4 * grp + r);
                if (d < a.dk) s_out[cv + d * pitch] = S[n][r];
            }
}

// The start of every segment: S_{s+1} = M_s S_s + N_s, in place of N_s.  A workgroup per (sequence, value head, 16 columns), a wave
// per 16 rows (two for dk > 128), on the fp32 matrix instructions; S_s goes round through LDS (by columns: a lane's four rows are one
// piece; two buffers, one barrier a step), M of the next two segments is on its way while one is multiplied.  A step is 0.6 us at
// dk = 64 and 2.6 at 128, where it reads 64 KB of M.  KT = dk / 16 rounded up; VEC: dk is a multiple of 4 (rows of M in 16-byte
// pieces).
template <int KT, bool VEC>
MP_KERNEL __launch_bounds__(KT <= 4 ? 256 : 512) void mp_delta_join(DeltaArgs a, DeltaPlan plan, int ncol) {
    constexpr int NT = (KT + 7) / 8, TH = KT <= 4 ? 256 : 512;
    constexpr bool kAhead = KT <= 8;              // (both would not fit the registers)
    __shared__ __align__(16) float St[2][16][16 * KT + 4];        // [column][row]
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, grp = lane >> 4, wave = tid >> 6;
    const int head = blockIdx.x % (a.B * a.Hv), ct = blockIdx.x / (a.B * a.Hv), b = head / a.Hv;      // (a head's workgroups, which read the same M, on one XCD
                                                                                                    //  where the heads are a multiple of 8)
    const int cv = 16 * ct + col, cc = min(cv, a.dv - 1);
    // segments behind which another one begins; the first one's N is its end state
    const int n = min(plan.nseg - 1, (length_of(a.lengths, b, a.T) + plan.len * kC - 1) / (plan.len * kC) - 1);
    float* N = plan.N + (size_t)head * (plan.nseg - 1) * a.dk * a.dv;
    const float* M = plan.M + (size_t)head * (plan.nseg - 1) * a.dk * a.dk;
    if (n < 2) return;
    for (int d = tid >> 4; d < 16 * KT; d += TH / 16) {
        St[0][tid & 15][d] = d < a.dk ? N[(size_t)d * a.dv + min(16 * ct + (tid & 15), a.dv - 1)] : 0.f;
        St[1][tid & 15][d] = 0.f;
    }
    float4 m[kAhead ? 2 : 1][NT][KT];
    f32x4 an[kAhead ? 2 : 1][NT];
    auto fetch = [&](int s, float4 (&mn)[NT][KT], f32x4 (&nn)[NT]) {
        const float* Ms = M + (size_t)s * a.dk * a.dk;
        const float* Ns = N + (size_t)s * a.dk * a.dv;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int row = min(16 * (wave + 8 * t) + col, a.dk - 1);
#pragma unroll
            for (int k = 0; k < KT; ++k) {
                const int d = 16 * k + 4 * grp;
                const float* p = Ms + (size_t)row * a.dk;
                if (VEC) mn[t][k] = *(const float4*)(p + (d < a.dk ? d : 0));      // (what is read behind dk meets zeros)
                else mn[t][k] = {p[min(d, a.dk - 1)], p[min(d + 1, a.dk - 1)], p[min(d + 2, a.dk - 1)], p[min(d + 3, a.dk - 1)]};
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) nn[t][r] = Ns[(size_t)min(16 * (wave + 8 * t) + 4 * grp + r, a.dk - 1) * a.dv + cc];
        }
    };
    auto step = [&](int s, float4 (&ms)[NT][KT], f32x4 (&acc)[NT]) {
        __syncthreads();
        const float (*const from)[16 * KT + 4] = St[(s - 1) & 1];
        float (*const to)[16 * KT + 4] = St[s & 1];
        float4 x[KT];
#pragma unroll
        for (int k = 0; k < KT; ++k) x[k] = *(const float4*)&from[col][16 * k + 4 * grp];      // (zeros behind dk)
        f32x4 odd[NT] = {};                                       // (a second chain of sums: a product does not wait for the one before it)
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                if (k & 1) odd[t] = mfma4(ms[t][k], x[k], odd[t]);
                else acc[t] = mfma4(ms[t][k], x[k], acc[t]);
            }
        // (no branches: what a lane has behind the last row or column is that row's or column's value once more)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            acc[t] += odd[t];
            const int d = 16 * (wave + 8 * t) + 4 * grp;
            if (16 * (wave + 8 * t) < 16 * KT)
                *(float4*)&to[col][d] = {d < a.dk ? acc[t][0] : 0.f, d + 1 < a.dk ? acc[t][1] : 0.f, d + 2 < a.dk ? acc[t][2] : 0.f, d + 3 < a.dk ? acc[t][3] : 0.f};
#pragma unroll
            for (int r = 0; r < 4; ++r) N[((size_t)s * a.dk + min(d + r, a.dk - 1)) * a.dv + cc] = acc[t][r];
        }
    };
    if constexpr (kAhead) {
        fetch(1, m[0], an[0]);
        __builtin_amdgcn_sched_barrier(0);                        // (in this order: the loop waits for as many as are older)
        fetch(min(2, n - 1), m[1], an[1]);
        __builtin_amdgcn_sched_barrier(0);
        int s = 1;
        for (; s + 1 < n; s += 2) {
            step(s, m[0], an[0]);
            fetch(min(s + 2, n - 1), m[0], an[0]);
            step(s + 1, m[1], an[1]);
            fetch(min(s + 3, n - 1), m[1], an[1]);
        }
        if (s < n) step(s, m[0], an[0]);
    } else {
        for (int s = 1; s < n; ++s) {
            fetch(s, m[0], an[0]);
            step(s, m[0], an[0]);
        }
    }
}

// Segments: as many as give the first pass two workgroups a CU, at least four chunks each; from four segments on they win (3 x the
// work in 2 / segments of the steps): 1 x 384 frames (three), 4 heads of 64, bf16 30.0 -> 31.3 us (fp32 41.9 -> 39.1), 1 x 512 36.3 -> 31.7
// (51.7 -> 39.9), 1 x 3000 166 -> 46 (248 -> 56), 1 x 32768 1683 -> 129 (2566 -> 162).  Where that makes no more than eight, and two
// workgroups of this kernel share a CU, twice as many: 2 x 4096, 32 heads of 64, bf16 160 -> 147 (fp32 247 -> 229), 4 x 4096, 16 heads of
// 128, bf16 347 -> 350 (fp32, one a CU, 597 -> 645); with more the join, whose steps are one after the other, takes what the passes
// gain (1 x 32768, 4 heads, 129 -> 160, fp32 162 -> 190).
static DeltaPlan plan_of(int B, int T, int Hv, int dk, int dv, bool two) {
    DeltaPlan p = {1, (T + kC - 1) / kC, nullptr, nullptr, nullptr};
    const long per = (long)B * Hv * ((dv + 63) / 64 + (dk + 63) / 64);
    const int nchunk = p.len, want = (int)min((long)nchunk / 4, (two && 512 / per <= 8 ? 1024 : 512) / per);
    if (want >= 4) {
        p.len = (nchunk + want - 1) / want;
        p.nseg = (nchunk + p.len - 1) / p.len;
    }
    return p;
}
static size_t prep_floats(int B, int T, int Hv) { return (size_t)B * Hv * ((T + kC - 1) / kC) * (kWsUnit / 4); }
size_t delta_ws_floats(int B, int T, int Hv, int dk, int dv) {
    const size_t cuts = max(plan_of(B, T, Hv, dk, dv, false).nseg, plan_of(B, T, Hv, dk, dv, true).nseg) - 1;
    return prep_floats(B, T, Hv) + (size_t)B * Hv * (cuts * dk * (dk + dv) + (cuts ? (size_t)dk * dv : 0)) + 4;
}

template <class E, int NK, int MODE, bool OUT>
static bool scan_pass(const DeltaArgs& a, const DeltaPlan& p, hipStream_t s) {
    constexpr int bytes = ScanLds<E, NK>::kBytes;
    static_assert(bytes <= 160 * 1024, "LDS of a CU");
    // (an attribute of the function on the current device: set at every launch, a call may come from any device's handle)
    if (bytes > 64 * 1024 && hipFuncSetAttribute((const void*)mp_delta_scan<E, NK, MODE, OUT>, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) return false;
    const int ncol = (a.dv + 63) / 64, ncolm = OUT ? 0 : (a.dk + 63) / 64, units = a.B * a.Hk * (OUT ? p.nseg : p.nseg - 1);
    hipLaunchKernelGGL((mp_delta_scan<E, NK, MODE, OUT>), dim3((unsigned)((units + 7) / 8 * 8 * (a.Hv / a.Hk) * (ncol + ncolm))), dim3(256), bytes, s, a, p, ncol, ncolm);
    return true;
}
template <class E, int NK, int MODE>
static bool scan_for(const DeltaArgs& a, hipStream_t s) {
    DeltaPlan p = plan_of(a.B, a.T, a.Hv, a.dk, a.dv, two_per_cu<E, NK>());
    if (p.nseg > 1) {
        p.N = a.ws + prep_floats(a.B, a.T, a.Hv);
        p.M = p.N + ((size_t)a.B * a.Hv * (p.nseg - 1) * a.dk * a.dv + 3) / 4 * 4;
        p.S0 = p.M + (size_t)a.B * a.Hv * (p.nseg - 1) * a.dk * a.dk;
        if (!scan_pass<E, NK, MODE, false>(a, p, s)) return false;
        const int ncol = (a.dv + 15) / 16;
        const dim3 grid((unsigned)(a.B * a.Hv * ncol));
        if (a.dk % 4) {
            if (a.dk <= 64) hipLaunchKernelGGL((mp_delta_join<4, false>), grid, dim3(256), 0, s, a, p, ncol);
            else if (a.dk <= 128) hipLaunchKernelGGL((mp_delta_join<8, false>), grid, dim3(512), 0, s, a, p, ncol);
            else hipLaunchKernelGGL((mp_delta_join<16, false>), grid, dim3(512), 0, s, a, p, ncol);
        } else {
            if (a.dk <= 64) hipLaunchKernelGGL((mp_delta_join<4, true>), grid, dim3(256), 0, s, a, p, ncol);
            else if (a.dk <= 128) hipLaunchKernelGGL((mp_delta_join<8, true>), grid, dim3(512), 0, s, a, p, ncol);
            else hipLaunchKernelGGL((mp_delta_join<16, true>), grid, dim3(512), 0, s, a, p, ncol);
        }
    }
    return scan_pass<E, NK, MODE, true>(a, p, s);
}
template <class E, int MODE>
static bool launch_mode(const DeltaArgs& a, hipStream_t s) {
    if (a.nchunk) {
        const dim3 grid((unsigned)(a.B * a.Hk * a.nchunk));
        constexpr int wide = Arith<E>::P == 1 ? 4 : 2;
        if (a.dk > 64) hipLaunchKernelGGL((mp_delta_prep<E, MODE, wide>), grid, dim3(64), 0, s, a);
        else hipLaunchKernelGGL((mp_delta_prep<E, MODE, 2>), grid, dim3(64), 0, s, a);
    }
    if (MODE == 2) return scan_for<E, 8, MODE>(a, s);
    constexpr int M = MODE == 2 ? 1 : MODE;
    const int nk = (a.dk + 31) / 32;
    return nk == 1 ? scan_for<E, 1, M>(a, s) : nk == 2 ? scan_for<E, 2, M>(a, s) : nk == 3 ? scan_for<E, 3, M>(a, s) : nk == 4 ? scan_for<E, 4, M>(a, s)
         : nk <= 6 ? scan_for<E, 6, M>(a, s) : scan_for<E, 8, M>(a, s);
}
template <class E>
static bool launch_for(const DeltaArgs& a, hipStream_t s) {
    const bool ok = a.dk < 8 || a.dv < 8 ? launch_mode<E, 2>(a, s) : a.dk % 8 ? launch_mode<E, 1>(a, s) : launch_mode<E, 0>(a, s);
    return hipGetLastError() == hipSuccess && ok;
}
bool launch_delta(const DeltaArgs& a, int dtype, hipStream_t s) {
    return dtype == kBF16 ? launch_for<bf16raw>(a, s) : launch_for<float>(a, s);
}

// ---------------------------------------------------------------- one frame per stream
// A workgroup owns (stream, value head, tile of columns): its part of the state is read once into registers -- a thread holds
// VEC columns of NR rows --, S^T k and S^T q are reduced together (o = e^g S^T q + (k . q) u needs no second pass), and the updated
// state is written once.  HBM-bound: 8 dk dv bytes per stream and head (512 streams, 16 heads of 128 x 128: 217 us, 4.94 TB/s, on one
// set of states or on six in turn; a copy reaches 5.08).  With slots a stream looks through those of the streams before it, whose
// number's square is nothing to 2048 streams (4 heads of 64 x 64: 48 us) and half of the call at 65536 (1.6 -> 3.5 ms).
template <class E, int VEC, int NR>
MP_KERNEL __launch_bounds__(256) void mp_delta_online(DeltaOnlineArgs a, int ntile, int log_lanes) {
    extern __shared__ float tick_lds[];               // k [dk] | q [dk] | partial sums [4 waves][2][lanes * VEC]
    const int tid = threadIdx.x, lanes = 1 << log_lanes, cl = tid & (lanes - 1), rl = tid >> log_lanes, rows = 256 >> log_lanes;
    const int ct = blockIdx.x % ntile, hv = blockIdx.x / ntile % a.Hv, st = blockIdx.x / ntile / a.Hv;
    const int hk = hv / (a.Hv / a.Hk);
    const int c0 = (ct * lanes + cl) * VEC;
    const bool cok = c0 < a.dv;
    const long slot = a.slots ? a.slots[st] : st;
    E* o = (E*)a.o + ((size_t)st * a.Hv + hv) * a.dv;
    if (slot < 0) {                              // no frame for this stream: an empty row, no state touched
        if (cok && rl == 0)
            for (int i = 0; i < VEC; ++i) store_f(o + c0 + i, 0.f);
        return;
    }
    // a row of the state that an earlier stream of this call uses, or that is not there: never plausible numbers
    bool refuse = slot >= a.n_slots;
    float* state = a.state + ((size_t)(refuse ? 0 : slot) * a.Hv + hv) * a.dk * a.dv;
    const E* v = (const E*)a.v + st * a.sv[0] + hv * a.sv[1];      // (requested with the state: a latency less behind the sums)
    float vc[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) vc[i] = load_f(v + min(c0, a.dv - VEC) + i);
    const float g = a.g[st * a.sg[0] + hv * a.sg[1]], beta = a.beta[st * a.sb[0] + hv * a.sb[1]];
    float S[NR][VEC];
    const float* const at = state + min(c0, a.dv - VEC);
#pragma unroll
    for (int n = 0; n < NR; ++n) {
        const int d = n * rows + rl;
        const float* x = at + (size_t)min(d, a.dk - 1) * a.dv;     // (no branch around the load: the rows behind dk are not used)
        if (VEC == 4) __builtin_memcpy(S[n], __builtin_assume_aligned(x, 16), 16);
        else S[n][0] = *x;
    }
    if (a.slots) {
        bool twice = false;
        for (int i = tid; i < st; i += 256) twice |= a.slots[i] == slot;
        refuse |= __syncthreads_or(twice) != 0;
    }
    float *lk = tick_lds, *lq = lk + a.dk, *part = lq + a.dk;
    const E* q = (const E*)a.q + st * a.sq[0] + hk * a.sq[1];
    const E* k = (const E*)a.k + st * a.sk[0] + hk * a.sk[1];
    for (int d = tid; d < a.dk; d += 256) { lk[d] = load_f(k + d); lq[d] = load_f(q + d); }
    const float eg = expf(g);
    __syncthreads();
    float ak[VEC], aq[VEC];
    for (int i = 0; i < VEC; ++i) ak[i] = aq[i] = 0.f;
#pragma unroll
    for (int n = 0; n < NR; ++n) {
        const int d = n * rows + rl;
        if (d < a.dk) {
            const float kd = lk[d], qd = lq[d];
#pragma unroll
            for (int i = 0; i < VEC; ++i) { ak[i] = fmaf(S[n][i], kd, ak[i]); aq[i] = fmaf(S[n][i], qd, aq[i]); }
        }
    }
    for (int m = lanes; m < 64; m <<= 1)
        for (int i = 0; i < VEC; ++i) { ak[i] += __shfl_xor(ak[i], m); aq[i] += __shfl_xor(aq[i], m); }
    const int wave = tid >> 6, cw = lanes * VEC;
    if ((tid & 63) < lanes)
        for (int i = 0; i < VEC; ++i) {
            part[(wave * 2 + 0) * cw + cl * VEC + i] = ak[i];
            part[(wave * 2 + 1) * cw + cl * VEC + i] = aq[i];
        }
    float kq = 0.f;
    for (int d = tid & 63; d < a.dk; d += 64) kq = fmaf(lk[d], lq[d], kq);
    for (int m = 1; m < 64; m <<= 1) kq += __shfl_xor(kq, m);
    __syncthreads();
    if (!cok) return;
    float u[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        float sk = 0.f, sq = 0.f;
        for (int w = 0; w < 4; ++w) {
            sk += part[(w * 2 + 0) * cw + cl * VEC + i];
            sq += part[(w * 2 + 1) * cw + cl * VEC + i];
        }
        u[i] = beta * (vc[i] - eg * sk);
        if (rl == 0) store_f(o + c0 + i, refuse ? __builtin_nanf("") : a.scale * (eg * sq + kq * u[i]));
    }
    if (refuse) return;
#pragma unroll
    for (int n = 0; n < NR; ++n) {
        const int d = n * rows + rl;
        if (d >= a.dk) continue;
        const float kd = lk[d];
        if (VEC == 4) {
            float4 x;
            x.x = fmaf(kd, u[0], eg * S[n][0]);
            x.y = fmaf(kd, u[VEC > 1 ? 1 : 0], eg * S[n][VEC > 1 ? 1 : 0]);
            x.z = fmaf(kd, u[VEC > 2 ? 2 : 0], eg * S[n][VEC > 2 ? 2 : 0]);
            x.w = fmaf(kd, u[VEC > 3 ? 3 : 0], eg * S[n][VEC > 3 ? 3 : 0]);
            *(float4*)(state + (size_t)d * a.dv + c0) = x;
        } else {
            state[(size_t)d * a.dv + c0] = fmaf(kd, u[0], eg * S[n][0]);
        }
    }
}

// 8 .. 32 threads side by side in a row of the state; 64 where they hold single columns: a row that two workgroups share is
// written in parts of cache lines (77 streams, 6 heads of 96 x 41: 8.6 us against 12.0 with 32, 14.2 with 16) -- up to dk = 128,
// where a thread holds 32 rows
static bool online_vec(const DeltaOnlineArgs& a) { return a.dv % 4 == 0 && (uintptr_t)a.state % 16 == 0; }
static int online_log_lanes(const DeltaOnlineArgs& a, int vec) {
    int lg = 3;
    while (lg < (vec == 1 && a.dk <= 128 ? 6 : 5) && (1 << lg) < (a.dv + vec - 1) / vec) ++lg;
    return lg;
}
static int online_tiles(const DeltaOnlineArgs& a, int vec, int lg) { return (int)((((int64_t)a.dv + vec - 1) / vec + (1 << lg) - 1) >> lg); }
int64_t delta_online_blocks(const DeltaOnlineArgs& a) {
    const int vec = online_vec(a) ? 4 : 1;
    return (int64_t)a.S * a.Hv * online_tiles(a, vec, online_log_lanes(a, vec));
}
template <class E, int VEC>
static void online_for(const DeltaOnlineArgs& a, hipStream_t s) {
    const int lg = online_log_lanes(a, VEC), ntile = online_tiles(a, VEC, lg), rows = 256 >> lg, nr = (a.dk + rows - 1) / rows;
    const size_t lds = (2 * (size_t)a.dk + 8 * (size_t)(VEC << lg)) * sizeof(float);
    const dim3 grid((unsigned)((size_t)a.S * a.Hv * ntile)), block(256);
    if (nr <= 2) hipLaunchKernelGGL((mp_delta_online<E, VEC, 2>), grid, block, lds, s, a, ntile, lg);
    else if (nr <= 4) hipLaunchKernelGGL((mp_delta_online<E, VEC, 4>), grid, block, lds, s, a, ntile, lg);
    else if (nr <= 8) hipLaunchKernelGGL((mp_delta_online<E, VEC, 8>), grid, block, lds, s, a, ntile, lg);
    else if (nr <= 16) hipLaunchKernelGGL((mp_delta_online<E, VEC, 16>), grid, block, lds, s, a, ntile, lg);
    else hipLaunchKernelGGL((mp_delta_online<E, VEC, 32>), grid, block, lds, s, a, ntile, lg);
}
bool launch_delta_online(const DeltaOnlineArgs& a, int dtype, hipStream_t s) {
    const bool vec = online_vec(a);
    if (dtype == kBF16) { if (vec) online_for<bf16raw, 4>(a, s); else online_for<bf16raw, 1>(a, s); }
    else { if (vec) online_for<float, 4>(a, s); else online_for<float, 1>(a, s); }
    return hipGetLastError() == hipSuccess;
}

}  // namespace mpseq
