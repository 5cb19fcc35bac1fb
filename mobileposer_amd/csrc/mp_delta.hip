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
// A value that is not finite reaches the frames behind it only, as in the recurrence: where a right-hand side holds one, the
// rows from there on are taken out of the products (0 * NaN in a triangular matrix's zeros would reach the frames before it)
// and their outputs and the column's state are NaN.
#include "mp_seq.h"

namespace mpseq {

constexpr int kC = 32;                            // frames per chunk
// workspace of one (sequence, value head, chunk), floats: T = (I + A)^{-1} and P = scale tril(Q K^T) o D as three 16 x 16 tiles
// (0,0), (1,0), (1,1) each, in the order in which a lane of v_mfma_f32_16x16x4_f32 takes its A operand
// ([tile][lane][4]: row lane & 15, columns 4 (lane >> 4) .. +3), then beta_i, e^{G_i}, e^{G_C - G_i}
constexpr int kTile = 256;
constexpr int kWsP = 3 * kTile, kWsBeta = 6 * kTile, kWsEg = kWsBeta + kC, kWsTail = kWsEg + kC, kWsUnit = kWsTail + kC;

size_t delta_ws_floats(int B, int T, int Hv) { return (size_t)B * Hv * ((T + kC - 1) / kC) * kWsUnit; }

static __device__ __forceinline__ int length_of(const int* lengths, int b, int T) {
    if (!lengths) return T;
    const int n = lengths[b];
    return n < 0 ? 0 : n > T ? T : n;
}
static __device__ __forceinline__ float clamp_g(float g) { return g < -1e4f ? -1e4f : g; }      // (NaN stays NaN)
static __device__ __forceinline__ bool not_finite(float x) { return !(fabsf(x) <= 3.402823466e38f); }

// 16 x 16 tile of X Y^T over dk: X rows x0 + l%16, Y rows y0 + l%16 of one head; any order of k serves as long as both take it
template <class E>
static __device__ __forceinline__ float4 row4(const E* p, int d, int dk, bool on) {
    float4 r;
    r.x = on && d + 0 < dk ? load_f(p + d + 0) : 0.f;
    r.y = on && d + 1 < dk ? load_f(p + d + 1) : 0.f;
    r.z = on && d + 2 < dk ? load_f(p + d + 2) : 0.f;
    r.w = on && d + 3 < dk ? load_f(p + d + 3) : 0.f;
    return r;
}
static __device__ __forceinline__ f32x4 mfma4(float4 a, float4 b, f32x4 c) {
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.x, b.x, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.y, b.y, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.z, b.z, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a.w, b.w, c, 0, 0, 0);
}

// One wave per (sequence, key head, chunk): K K^T and Q K^T once, then the value heads that share the key head.
template <class E>
MP_KERNEL __launch_bounds__(64) void mp_delta_prep(DeltaArgs a) {
    __shared__ float A[kC][kC + 1];
    const int unit = blockIdx.x, c = unit % a.nchunk, hk = unit / a.nchunk % a.Hk, b = unit / a.nchunk / a.Hk;
    const int lane = threadIdx.x, col = lane & 15, grp = lane >> 4, t0 = c * kC;
    const int len = length_of(a.lengths, b, a.T);
    if (t0 >= len) return;
    const E* q = (const E*)a.q + b * a.sq[0] + hk * a.sq[2];
    const E* k = (const E*)a.k + b * a.sk[0] + hk * a.sk[2];
    f32x4 kk[3] = {}, qk[3] = {};
    for (int d = 4 * grp; d - 4 * grp < a.dk; d += 16) {
        float4 fk[2], fq[2];
        for (int I = 0; I < 2; ++I) {
            const int t = t0 + 16 * I + col;
            const bool on = t < len;
            fk[I] = row4(k + (on ? t : 0) * a.sk[1], d, a.dk, on);
            fq[I] = row4(q + (on ? t : 0) * a.sq[1], d, a.dk, on);
        }
        kk[0] = mfma4(fk[0], fk[0], kk[0]);
        kk[1] = mfma4(fk[1], fk[0], kk[1]);
        kk[2] = mfma4(fk[1], fk[1], kk[2]);
        qk[0] = mfma4(fq[0], fk[0], qk[0]);
        qk[1] = mfma4(fq[1], fk[0], qk[1]);
        qk[2] = mfma4(fq[1], fk[1], qk[2]);
    }
    const int rep = a.Hv / a.Hk;
    for (int e = 0; e < rep; ++e) {
        const int hv = hk * rep + e;
        float* ws = a.ws + ((size_t)(b * a.Hv + hv) * a.nchunk + c) * kWsUnit;
        const int i = lane & 31, t = t0 + i;
        const bool on = t < len;
        const float beta = on ? a.beta[b * a.sb[0] + t * a.sb[1] + hv * a.sb[2]] : 0.f;
        double G = on ? (double)clamp_g(a.g[b * a.sg[0] + t * a.sg[1] + hv * a.sg[2]]) : 0.0;
        for (int s = 1; s < kC; s <<= 1) {
            const double up = __shfl_up(G, s, 32);
            if (i >= s) G += up;
        }
        const double last = __shfl(G, kC - 1, 32);
        if (lane < kC) {
            ws[kWsBeta + i] = beta;
            ws[kWsEg + i] = expf((float)G);
            ws[kWsTail + i] = expf((float)(last - G));
        }
        // D layout of an accumulator: row 4 grp + r, column col
        for (int tile = 0; tile < 3; ++tile) {
            const int I = tile > 0, J = tile > 1;
            const double Gj = __shfl(G, 16 * J + col, 64);
            for (int r = 0; r < 4; ++r) {
                const int ri = 16 * I + 4 * grp + r, cj = 16 * J + col;
                const float D = expf((float)(__shfl(G, ri, 64) - Gj));
                const float bi = __shfl(beta, ri, 64);
                A[ri][cj] = cj < ri ? bi * D * kk[tile][r] : 0.f;
                // P in operand order: lane (row & 15) + 16 (column / 4 within the tile), element column % 4
                ws[kWsP + tile * kTile + ((ri & 15) + 16 * (col >> 2)) * 4 + (col & 3)] = cj <= ri ? a.scale * D * qk[tile][r] : 0.f;
            }
        }
        __syncthreads();
        // T = (I + A)^{-1} by forward substitution, lane = column
        float x[kC];
        for (int n = 0; n < kC; ++n) {
            float s = n == i ? 1.f : 0.f;
            for (int j = 0; j < n; ++j) s -= j < i ? 0.f : A[n][j] * x[j];
            x[n] = n < i ? 0.f : s;
        }
        if (lane < kC) {
            const int J = i >> 4, cc = i & 15;
            for (int n = 0; n < kC; ++n) {
                const int I = n >> 4;
                if (I >= J) ws[(I + J) * kTile + ((n & 15) + 16 * (cc >> 2)) * 4 + (cc & 3)] = x[n];
            }
        }
        __syncthreads();
    }
}

// One wave per (sequence, value head, 16 columns of the state): the walk over the chunks.  NK = dk / 16 rounded up.
// The accumulator layout (row 4 grp + r, column col) of a tile IS the B operand of four v_mfma_f32_16x16x4_f32 when their k
// slots are taken as rows 4 grp + r of step r, so the state, the right-hand sides and U never leave their registers.
template <class E, int NK>
MP_KERNEL __launch_bounds__(64) void mp_delta_scan(DeltaArgs a, int ncol) {
    const int lane = threadIdx.x, col = lane & 15, grp = lane >> 4;
    const int ct = blockIdx.x % ncol, hv = blockIdx.x / ncol % a.Hv, b = blockIdx.x / ncol / a.Hv;
    const int hk = hv / (a.Hv / a.Hk);
    const int cv = 16 * ct + col;
    const bool cok = cv < a.dv;
    const int len = length_of(a.lengths, b, a.T);
    const E* q = (const E*)a.q + b * a.sq[0] + hk * a.sq[2];
    const E* k = (const E*)a.k + b * a.sk[0] + hk * a.sk[2];
    const E* v = (const E*)a.v + b * a.sv[0] + hv * a.sv[2] + cv;
    E* o = (E*)a.o + ((size_t)b * a.T * a.Hv + hv) * a.dv + cv;
    const size_t so = (size_t)a.Hv * a.dv;
    const size_t sbase = (size_t)(b * a.Hv + hv) * a.dk * a.dv + cv;
    f32x4 S[NK];
#pragma unroll
    for (int n = 0; n < NK; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int d = 16 * n + 4 * grp + r;
            S[n][r] = a.s_in && cok && d < a.dk ? a.s_in[sbase + (size_t)d * a.dv] : 0.f;
        }
    const float nan = __builtin_nanf("");
    for (int c = 0; c * kC < len; ++c) {
        const float* ws = a.ws + ((size_t)(b * a.Hv + hv) * a.nchunk + c) * kWsUnit;
        const int t0 = c * kC;
        f32x4 ks[2] = {}, qs[2] = {};
#pragma unroll
        for (int n = 0; n < NK; ++n) {
            const float4 s4 = {S[n][0], S[n][1], S[n][2], S[n][3]};
            for (int I = 0; I < 2; ++I) {
                const int t = t0 + 16 * I + col;
                const bool on = t < len;
                ks[I] = mfma4(row4(k + (on ? t : 0) * a.sk[1], 16 * n + 4 * grp, a.dk, on), s4, ks[I]);
                qs[I] = mfma4(row4(q + (on ? t : 0) * a.sq[1], 16 * n + 4 * grp, a.dk, on), s4, qs[I]);
            }
        }
        float4 R[2];
        bool bad = false;
        for (int I = 0; I < 2; ++I) {
            float rr[4];
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * I + 4 * grp + r, t = t0 + i;
                const float vv = cok && t < len ? load_f(v + (size_t)t * a.sv[1]) : 0.f;
                rr[r] = ws[kWsBeta + i] * (vv - ws[kWsEg + i] * ks[I][r]);
                bad |= not_finite(rr[r]);
            }
            R[I] = {rr[0], rr[1], rr[2], rr[3]};
        }
        int first = kC;                                            // this column's first row that is not finite
        const bool any_bad = __any(bad);
        if (any_bad) {
            for (int I = 1; I >= 0; --I)
                for (int r = 3; r >= 0; --r)
                    if (not_finite(((const float*)&R[I])[r])) first = 16 * I + 4 * grp + r;
            first = min(first, __shfl_xor(first, 16));
            first = min(first, __shfl_xor(first, 32));
            for (int I = 0; I < 2; ++I)
                for (int r = 0; r < 4; ++r)
                    if (16 * I + 4 * grp + r >= first) ((float*)&R[I])[r] = 0.f;
        }
        const float4* T4 = (const float4*)ws;
        const float4* P4 = (const float4*)(ws + kWsP);
        f32x4 u[2] = {}, w[2] = {};
        u[0] = mfma4(T4[lane], R[0], u[0]);
        u[1] = mfma4(T4[64 + lane], R[0], u[1]);
        u[1] = mfma4(T4[128 + lane], R[1], u[1]);
        if (any_bad)
            for (int I = 0; I < 2; ++I)
                for (int r = 0; r < 4; ++r)
                    if (16 * I + 4 * grp + r >= first) u[I][r] = 0.f;
        const float4 u0 = {u[0][0], u[0][1], u[0][2], u[0][3]}, u1 = {u[1][0], u[1][1], u[1][2], u[1][3]};
        w[0] = mfma4(P4[lane], u0, w[0]);
        w[1] = mfma4(P4[64 + lane], u0, w[1]);
        w[1] = mfma4(P4[128 + lane], u1, w[1]);
        for (int I = 0; I < 2; ++I)
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * I + 4 * grp + r, t = t0 + i;
                float ov = a.scale * ws[kWsEg + i] * qs[I][r] + w[I][r];
                if (i >= first) ov = nan;
                if (cok && t < len) store_f(o + (size_t)t * so, ov);
            }
        // S' = e^{G_C} S0 + K^T (e^{G_C - G} U)
        const float whole = ws[kWsEg + kC - 1];
        float4 ut[2];
        for (int I = 0; I < 2; ++I) {
            float x[4];
            for (int r = 0; r < 4; ++r) x[r] = ws[kWsTail + 16 * I + 4 * grp + r] * u[I][r];
            ut[I] = {x[0], x[1], x[2], x[3]};
        }
#pragma unroll
        for (int n = 0; n < NK; ++n) {
            S[n] *= whole;
            const int d = 16 * n + col;
            for (int I = 0; I < 2; ++I) {
                float kt[4];
                for (int r = 0; r < 4; ++r) {
                    const int t = t0 + 16 * I + 4 * grp + r;
                    kt[r] = d < a.dk && t < len ? load_f(k + (size_t)t * a.sk[1] + d) : 0.f;
                }
                S[n] = mfma4({kt[0], kt[1], kt[2], kt[3]}, ut[I], S[n]);
            }
            if (first < kC)
                for (int r = 0; r < 4; ++r) S[n][r] = nan;
        }
    }
    if (cok)
        for (int t = len + grp; t < a.T; t += 4) store_f(o + (size_t)t * so, 0.f);
    if (a.s_out && cok)
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int d = 16 * n + 4 * grp + r;
                if (d < a.dk) a.s_out[sbase + (size_t)d * a.dv] = S[n][r];
            }
}

template <class E, int NK>
static void scan_for(const DeltaArgs& a, hipStream_t s) {
    const int ncol = (a.dv + 15) / 16;
    hipLaunchKernelGGL((mp_delta_scan<E, NK>), dim3((unsigned)(a.B * a.Hv * ncol)), dim3(64), 0, s, a, ncol);
}
template <class E>
static bool launch_for(const DeltaArgs& a, hipStream_t s) {
    if (a.nchunk) hipLaunchKernelGGL(mp_delta_prep<E>, dim3((unsigned)(a.B * a.Hk * a.nchunk)), dim3(64), 0, s, a);
    const int nk = (a.dk + 15) / 16;
    if (nk <= 2) scan_for<E, 2>(a, s);
    else if (nk <= 4) scan_for<E, 4>(a, s);
    else if (nk <= 8) scan_for<E, 8>(a, s);
    else scan_for<E, 16>(a, s);
    return hipGetLastError() == hipSuccess;
}
bool launch_delta(const DeltaArgs& a, int dtype, hipStream_t s) {
    return dtype == kBF16 ? launch_for<bf16raw>(a, s) : launch_for<float>(a, s);
}

// ---------------------------------------------------------------- one frame per stream
// A workgroup owns (stream, value head, tile of columns): its part of the state is read once into registers -- a thread holds
// VEC columns of NR rows --, S^T k and S^T q are reduced together (o = e^g S^T q + (k . q) u needs no second pass), and the updated
// state is written once.  HBM-bound: 8 dk dv bytes per stream and head.
template <class E, int VEC, int NR>
MP_KERNEL __launch_bounds__(256) void mp_delta_online(DeltaOnlineArgs a, int ntile, int log_lanes) {
    extern __shared__ float lds[];               // k [dk] | q [dk] | partial sums [4 waves][2][lanes * VEC]
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
    float S[NR][VEC];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
        const int d = n * rows + rl;
        if (VEC == 4) {
            float4 x = {0.f, 0.f, 0.f, 0.f};
            if (cok && d < a.dk) x = *(const float4*)(state + (size_t)d * a.dv + c0);
            S[n][0] = x.x; S[n][VEC > 1 ? 1 : 0] = x.y; S[n][VEC > 2 ? 2 : 0] = x.z; S[n][VEC > 3 ? 3 : 0] = x.w;
        } else {
            S[n][0] = cok && d < a.dk ? state[(size_t)d * a.dv + c0] : 0.f;
        }
    }
    if (a.slots) {
        bool twice = false;
        for (int i = tid; i < st; i += 256) twice |= a.slots[i] == slot;
        refuse |= __syncthreads_or(twice) != 0;
    }
    float *lk = lds, *lq = lds + a.dk, *part = lds + 2 * a.dk;
    const E* q = (const E*)a.q + st * a.sq[0] + hk * a.sq[1];
    const E* k = (const E*)a.k + st * a.sk[0] + hk * a.sk[1];
    for (int d = tid; d < a.dk; d += 256) { lk[d] = load_f(k + d); lq[d] = load_f(q + d); }
    const float eg = expf(a.g[st * a.sg[0] + hv * a.sg[1]]), beta = a.beta[st * a.sb[0] + hv * a.sb[1]];
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
    const E* v = (const E*)a.v + st * a.sv[0] + hv * a.sv[1];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        float sk = 0.f, sq = 0.f;
        for (int w = 0; w < 4; ++w) {
            sk += part[(w * 2 + 0) * cw + cl * VEC + i];
            sq += part[(w * 2 + 1) * cw + cl * VEC + i];
        }
        u[i] = beta * (load_f(v + c0 + i) - eg * sk);
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

template <class E, int VEC>
static void online_for(const DeltaOnlineArgs& a, hipStream_t s) {
    const int need = (a.dv + VEC - 1) / VEC;
    int lg = 3;                                  // 8 .. 32 threads side by side in a row of the state
    while (lg < 5 && (1 << lg) < need) ++lg;
    const int ntile = (need + (1 << lg) - 1) >> lg, rows = 256 >> lg, nr = (a.dk + rows - 1) / rows;
    const size_t lds = (2 * (size_t)a.dk + 8 * (size_t)(VEC << lg)) * sizeof(float);
    const dim3 grid((unsigned)((size_t)a.S * a.Hv * ntile)), block(256);
    if (nr <= 2) hipLaunchKernelGGL((mp_delta_online<E, VEC, 2>), grid, block, lds, s, a, ntile, lg);
    else if (nr <= 4) hipLaunchKernelGGL((mp_delta_online<E, VEC, 4>), grid, block, lds, s, a, ntile, lg);
    else if (nr <= 8) hipLaunchKernelGGL((mp_delta_online<E, VEC, 8>), grid, block, lds, s, a, ntile, lg);
    else if (nr <= 16) hipLaunchKernelGGL((mp_delta_online<E, VEC, 16>), grid, block, lds, s, a, ntile, lg);
    else hipLaunchKernelGGL((mp_delta_online<E, VEC, 32>), grid, block, lds, s, a, ntile, lg);
}
bool launch_delta_online(const DeltaOnlineArgs& a, int dtype, hipStream_t s) {
    const bool vec = a.dv % 4 == 0 && (uintptr_t)a.state % 16 == 0;
    if (dtype == kBF16) { if (vec) online_for<bf16raw, 4>(a, s); else online_for<bf16raw, 1>(a, s); }
    else { if (vec) online_for<float, 4>(a, s); else online_for<float, 1>(a, s); }
    return hipGetLastError() == hipSuccess;
}

}  // namespace mpseq
