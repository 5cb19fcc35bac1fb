// Entry points of the sequence operators (include/mobileposer_hip.h, "sequence operators"): argument checks on the host, then the
// launches of mp_delta.hip / mp_adapt.hip on the CALLER'S stream itself.  They touch nothing the handle owns -- no library stream,
// no workspace, no carried state: all memory is the caller's --, so calls on different streams do not wait for each other, a call
// can be captured into the caller's own graph, and a body-only handle serves them as well.
#include "mp_host.h"
#include "mp_seq.h"

namespace {

// A launch counts its threads in 32 bits: so many workgroups of 256 or of 64 threads.
constexpr int64_t kMaxBlocks = (1 << 24) - 1, kMaxBlocks64 = (1 << 26) - 1;

int bad_type(mp_handle* h, const char* what, int dtype) {
    return fail(h, MP_ERR_INVALID, "%s: dtype %d (MP_F32 = 0 or MP_BF16 = 1)", what, dtype);
}
bool heads_ok(int Hk, int Hv, int dk, int dv) { return Hk >= 1 && Hv >= 1 && Hv % Hk == 0 && dk >= 1 && dk <= 256 && dv >= 1; }

}  // namespace

extern "C" {

size_t mp_delta_rule_workspace(int B, int T, int Hv, int dk, int dv) {
    return B < 1 || T < 1 || Hv < 1 || dk < 1 || dv < 1 ? 0 : mpseq::delta_ws_floats(B, T, Hv, dk, dv) * sizeof(float);
}

int mp_delta_rule(mp_handle* h, int dtype, const void* q_dev, const void* k_dev, const void* v_dev, const float* g_dev,
                  const float* beta_dev, const int64_t strides[15], const int32_t* lengths_dev, int B, int T, int Hk, int Hv,
                  int dk, int dv, float scale, void* o_dev, const float* state_in_dev, float* state_out_dev, void* ws_dev,
                  size_t ws_bytes, void* stream) {
    if (!h) return MP_ERR_INVALID;
    if (dtype != mpseq::kF32 && dtype != mpseq::kBF16) return bad_type(h, "mp_delta_rule", dtype);
    if (B < 0 || T < 0 || !heads_ok(Hk, Hv, dk, dv))
        return fail(h, MP_ERR_INVALID, "mp_delta_rule: B = %d, T = %d, heads %d / %d, head sizes %d / %d (Hv a multiple of Hk, dk 1..256)", B, T, Hk, Hv, dk, dv);
    if (B == 0) return MP_OK;
    if (T > 0 && (!q_dev || !k_dev || !v_dev || !g_dev || !beta_dev || !strides || !o_dev))
        return fail(h, MP_ERR_INVALID, "mp_delta_rule: NULL buffer");
    const size_t need = mp_delta_rule_workspace(B, T, Hv, dk, dv);
    if (need && (!ws_dev || ws_bytes < need || (uintptr_t)ws_dev % 16))
        return fail(h, MP_ERR_INVALID, "mp_delta_rule: workspace of %zu bytes, %zu needed (16-byte aligned)", ws_bytes, need);
    const int64_t nchunk = ((int64_t)T + 31) / 32;
    if ((int64_t)B * Hk * nchunk > kMaxBlocks64 || ((int64_t)B * Hk + 7) * (Hv / Hk) * (((int64_t)dv + 63) / 64) > kMaxBlocks ||
        (int64_t)Hv * dv > (1 << 24) - 1)
        return fail(h, MP_ERR_INVALID, "mp_delta_rule: batch of %d x %d frames, %d heads is too large for one call", B, T, Hv);
    ON_DEVICE(h);
    mpseq::DeltaArgs a;
    memset(&a, 0, sizeof(a));
    a.q = q_dev; a.k = k_dev; a.v = v_dev; a.g = g_dev; a.beta = beta_dev;
    if (strides)
        for (int i = 0; i < 3; ++i) {
            // 32 frames are addressed with 32-bit byte offsets
            if (T > 1 && (strides[3 * i + 1] < 0 || strides[3 * i + 1] > (1 << 24) - 1))
                return fail(h, MP_ERR_INVALID, "mp_delta_rule: frame stride of %lld elements (0..2^24 - 1)", (long long)strides[3 * i + 1]);
            a.sq[i] = strides[i]; a.sk[i] = strides[3 + i]; a.sv[i] = strides[6 + i]; a.sg[i] = strides[9 + i]; a.sb[i] = strides[12 + i];
        }
    a.lengths = lengths_dev; a.B = B; a.T = T; a.Hk = Hk; a.Hv = Hv; a.dk = dk; a.dv = dv; a.scale = scale;
    a.o = o_dev; a.s_in = state_in_dev; a.s_out = state_out_dev; a.ws = (float*)ws_dev; a.nchunk = (int)nchunk;
    if (!mpseq::launch_delta(a, dtype, (hipStream_t)stream)) return fail(h, MP_ERR_HIP, "mp_delta_rule: launch failed");
    return MP_OK;
}

int mp_delta_rule_online(mp_handle* h, int dtype, const void* q_dev, const void* k_dev, const void* v_dev, const float* g_dev,
                         const float* beta_dev, const int64_t strides[10], const int32_t* slots_dev, int S, int n_slots, int Hk,
                         int Hv, int dk, int dv, float scale, void* o_dev, float* state_dev, void* stream) {
    if (!h) return MP_ERR_INVALID;
    if (dtype != mpseq::kF32 && dtype != mpseq::kBF16) return bad_type(h, "mp_delta_rule_online", dtype);
    if (S < 0 || n_slots < 0 || !heads_ok(Hk, Hv, dk, dv))
        return fail(h, MP_ERR_INVALID, "mp_delta_rule_online: %d streams on %d states, heads %d / %d, head sizes %d / %d (Hv a multiple of Hk, dk 1..256)",
                    S, n_slots, Hk, Hv, dk, dv);
    if (S == 0) return MP_OK;
    if (!q_dev || !k_dev || !v_dev || !g_dev || !beta_dev || !strides || !o_dev || !state_dev || n_slots < 1)
        return fail(h, MP_ERR_INVALID, "mp_delta_rule_online: NULL buffer or no state");
    if (!slots_dev && S > n_slots) return fail(h, MP_ERR_INVALID, "mp_delta_rule_online: %d streams on %d states without slots", S, n_slots);
    ON_DEVICE(h);
    mpseq::DeltaOnlineArgs a;
    a.q = q_dev; a.k = k_dev; a.v = v_dev; a.g = g_dev; a.beta = beta_dev;
    for (int i = 0; i < 2; ++i) {
        a.sq[i] = strides[i]; a.sk[i] = strides[2 + i]; a.sv[i] = strides[4 + i]; a.sg[i] = strides[6 + i]; a.sb[i] = strides[8 + i];
    }
    a.slots = slots_dev; a.S = S; a.n_slots = n_slots; a.Hk = Hk; a.Hv = Hv; a.dk = dk; a.dv = dv; a.scale = scale;
    a.o = o_dev; a.state = state_dev;
    if (mpseq::delta_online_blocks(a) > kMaxBlocks)
        return fail(h, MP_ERR_INVALID, "mp_delta_rule_online: %d streams of %d heads are too many for one call", S, Hv);
    if (!mpseq::launch_delta_online(a, dtype, (hipStream_t)stream)) return fail(h, MP_ERR_HIP, "mp_delta_rule_online: launch failed");
    return MP_OK;
}

size_t mp_linear_adapted_workspace(int B, int T, int r) {
    return B < 1 || T < 1 || r < 1 ? 0 : mpseq::adapt_ws_floats(B, T, r) * sizeof(float);
}

int mp_linear_adapted(mp_handle* h, int dtype, const void* x_dev, const int64_t strides[2], const void* w_dev, const void* bias_dev,
                      const void* down_dev, const void* up_dev, const float* scale_dev, const int32_t* ids_dev, int B, int T, int K,
                      int M, int n_adapters, int r, int relu, void* y_dev, void* ws_dev, size_t ws_bytes, void* stream) {
    if (!h) return MP_ERR_INVALID;
    if (dtype != mpseq::kF32 && dtype != mpseq::kBF16) return bad_type(h, "mp_linear_adapted", dtype);
    if (B < 0 || T < 0 || K < 1 || M < 1 || n_adapters < 1 || r < 1 || r > 128)
        return fail(h, MP_ERR_INVALID, "mp_linear_adapted: B = %d, T = %d, %d -> %d, %d adapters of rank %d (rank 1..128)", B, T, K, M, n_adapters, r);
    if (B == 0 || T == 0) return MP_OK;
    if (!x_dev || !strides || !w_dev || !down_dev || !up_dev || !ids_dev || !y_dev)
        return fail(h, MP_ERR_INVALID, "mp_linear_adapted: NULL buffer");
    const size_t need = mp_linear_adapted_workspace(B, T, r);
    if (!ws_dev || ws_bytes < need || (uintptr_t)ws_dev % 16)
        return fail(h, MP_ERR_INVALID, "mp_linear_adapted: workspace of %zu bytes, %zu needed (16-byte aligned)", ws_bytes, need);
    if (!mpseq::adapt_fits(B, T, M, r))
        return fail(h, MP_ERR_INVALID, "mp_linear_adapted: %d x %d rows to %d columns are too many for one call", B, T, M);
    ON_DEVICE(h);
    mpseq::AdaptArgs a;
    a.x = x_dev; a.sx[0] = strides[0]; a.sx[1] = strides[1]; a.w = w_dev; a.ldw = K; a.bias = bias_dev; a.down = down_dev; a.up = up_dev;
    a.scale = scale_dev; a.ids = ids_dev; a.B = B; a.T = T; a.K = K; a.M = M; a.n = n_adapters; a.r = r; a.relu = relu != 0;
    a.y = y_dev; a.sy[0] = (long)T * M; a.sy[1] = M; a.ws = (float*)ws_dev;
    if (!mpseq::launch_adapt(a, dtype, (hipStream_t)stream)) return fail(h, MP_ERR_HIP, "mp_linear_adapted: launch failed");
    return MP_OK;
}

}  // extern "C"
