// A linear layer over the rows of many sequences with a low-rank adapter per sequence beside the shared weight:
//   y_n = act(W x_n + b + scale_a Up_a (Down_a x_n)),   a = ids[sequence of n]   (negative: the shared layer alone).
#include "mp_seq.h"

namespace mpseq {

size_t adapt_ws_floats(int B, int T, int r) { return (size_t)B * T * r; }

// z [row][r] = scale_a Down_a x_row: a wave per (row, component)
template <class E>
MP_KERNEL __launch_bounds__(256) void mp_adapt_down(AdaptArgs a, long total) {
    const long i = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= total) return;
    const int lane = threadIdx.x & 63, j = (int)(i % a.r);
    const long row = i / a.r;
    const int b = (int)(row / a.T), t = (int)(row % a.T), id = a.ids[b];
    float z = 0.f;
    if (id >= 0 && id < a.n) {
        const E* x = (const E*)a.x + b * a.sx[0] + t * a.sx[1];
        const E* d = (const E*)a.down + ((size_t)id * a.r + j) * a.K;
        for (int k = lane; k < a.K; k += 64) z = fmaf(load_f(x + k), load_f(d + k), z);
        for (int m = 1; m < 64; m <<= 1) z += __shfl_xor(z, m);
        if (a.scale) z *= a.scale[id];
    }
    if (lane == 0) a.ws[i] = z;
}

template <class E>
MP_KERNEL __launch_bounds__(256) void mp_adapt_rows(AdaptArgs a, long rows) {
    __shared__ float xs[16][17], wsh[16][17];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, m = blockIdx.y * 16 + tx;
    const long row = (long)blockIdx.x * 16 + ty;
    const bool rok = row < rows, mok = m < a.M;
    const int b = rok ? (int)(row / a.T) : 0, t = rok ? (int)(row % a.T) : 0;
    const E* x = (const E*)a.x + b * a.sx[0] + t * a.sx[1];
    const int wm = blockIdx.y * 16 + ty;
    const E* w = (const E*)a.w + (size_t)(wm < a.M ? wm : 0) * a.K;
    float acc = 0.f;
    for (int k0 = 0; k0 < a.K; k0 += 16) {
        const int k = k0 + tx;
        xs[ty][tx] = rok && k < a.K ? load_f(x + k) : 0.f;
        wsh[ty][tx] = wm < a.M && k < a.K ? load_f(w + k) : 0.f;
        __syncthreads();
        for (int j = 0; j < 16; ++j) acc = fmaf(xs[ty][j], wsh[tx][j], acc);
        __syncthreads();
    }
    if (!rok || !mok) return;
    if (a.bias) acc += load_f((const E*)a.bias + m);
    const int id = a.ids[b];
    if (id >= a.n) acc = __builtin_nanf("");
    else if (id >= 0) {
        const E* up = (const E*)a.up + ((size_t)id * a.M + m) * a.r;
        const float* z = a.ws + row * a.r;
        for (int j = 0; j < a.r; ++j) acc = fmaf(z[j], load_f(up + j), acc);
    }
    if (a.relu) acc = relu_(acc);
    store_f((E*)a.y + (size_t)row * a.M + m, acc);
}

template <class E>
static bool launch_for(const AdaptArgs& a, hipStream_t s) {
    const long rows = (long)a.B * a.T, total = rows * a.r;
    hipLaunchKernelGGL(mp_adapt_down<E>, dim3((unsigned)((total + 3) / 4)), dim3(256), 0, s, a, total);
    hipLaunchKernelGGL(mp_adapt_rows<E>, dim3((unsigned)((rows + 15) / 16), (unsigned)((a.M + 15) / 16)), dim3(256), 0, s, a, rows);
    return hipGetLastError() == hipSuccess;
}
bool launch_adapt(const AdaptArgs& a, int dtype, hipStream_t s) {
    return dtype == kBF16 ? launch_for<bf16raw>(a, s) : launch_for<float>(a, s);
}

}  // namespace mpseq
