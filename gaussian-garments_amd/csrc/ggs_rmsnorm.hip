// ggs_rmsnorm.hip -- root-mean-square norm over the channels of a feature map with the residual's addition, forward and
// backward: the pixel norm of StyleGAN-type networks (ggsplat.stylenet).  No reference counterpart.
//
// Layout [outer][C][inner]: element (o, c, i) at (o C + c) inner + i.  inner = H W for channels-first feature maps, 1 for rows
// of C contiguous values (style vectors, feature rows, channels-last maps).  A "pixel" below is one (o, i).
//
//   h = x + r,  q = 1 / sqrt(mean_c h_c^2 + eps),  n = q h,  y = w n
//   dL/dh = q (w gy - n mean_c(w gy n)) + gh,   dx = dr = dL/dh,   dw_c = sum over pixels of gy n
//
// Element types float, half, bfloat16 (computed in float) and double (in double).  The backward pass is given h itself in
// float and double; in 16 bits it is given x and r and adds them again, because the h that was stored is rounded to 8 or 11
// bits and dw, a sum over all pixels that may be a 32-bit tensor, would carry that rounding.  q is kept in the accumulation type.
// HBM-bound: forward reads x, r and writes y, h; backward reads h (x, r), gy, gh and writes dx: 8 elements a value at most.
#include "ggs_kernels.h"

namespace {

template <typename T> struct Acc { typedef float type; };
template <> struct Acc<double> { typedef double type; };

template <typename T> struct NormArgs {
    typedef typename Acc<T>::type A;
    size_t outer, inner;
    int C;
    const T *x, *r, *gy, *gh;
    const void* w;
    bool w32;                    // w (and dw) are float whatever T is
    A eps;
    T *y, *h, *dx;
    A* q;                        // [outer][inner]
    A* partial;                  // [n_partial][C]
    int n_partial;
    void* dw;
};

template <typename T> __device__ __forceinline__ typename Acc<T>::type weight(const NormArgs<T>& a, int c) {
    typedef typename Acc<T>::type A;
    if (!a.w) return (A)1;
    return a.w32 ? (A) static_cast<const float*>(a.w)[c] : (A) static_cast<const T*>(a.w)[c];
}
template <typename T> __device__ __forceinline__ typename Acc<T>::type value(const NormArgs<T>& a, size_t at) {
    typedef typename Acc<T>::type A;
    return a.r ? (A)a.x[at] + (A)a.r[at] : (A)a.x[at];
}

// Sum over the 4 waves of a workgroup, lane by lane.
template <typename A> __device__ __forceinline__ A sum_waves(A s, A* lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __syncthreads();
    lds[wave * 64 + lane] = s;
    __syncthreads();
    return (lds[lane] + lds[64 + lane]) + (lds[128 + lane] + lds[192 + lane]);
}
template <typename A> __device__ __forceinline__ A sum_lanes(A s) {
#pragma unroll
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
    return s;
}

// Any channel count, two passes over the data (the second one from the caches).  PLANES: 64 pixels of one map a workgroup, its
// four waves take every fourth channel; otherwise one row a workgroup.
template <typename T, bool PLANES>
__global__ __launch_bounds__(256) void k_rms_forward(NormArgs<T> a) {
    typedef typename Acc<T>::type A;
    __shared__ A lds[256];
    const size_t tiles = PLANES ? (a.inner + 63) / 64 : 1;
    const size_t o = blockIdx.x / tiles, i = PLANES ? (blockIdx.x % tiles) * 64 + (threadIdx.x & 63) : 0;
    const int c0 = PLANES ? threadIdx.x >> 6 : threadIdx.x, step = PLANES ? 4 : 256;
    const int C = i < a.inner ? a.C : 0;                            // lanes beyond the map only take part in the barriers
    const size_t base = o * a.C * a.inner + i;
    A s = 0;
    for (int c = c0; c < C; c += step) {
        const A h = value(a, base + c * a.inner);
        s += h * h;
    }
    if (!PLANES) s = sum_lanes(s);
    s = sum_waves<A>(s, lds);
    const A q = (A)1 / sqrt(s / (A)a.C + a.eps);
    if (c0 == 0 && a.q && i < a.inner) a.q[o * a.inner + i] = q;
    for (int c = c0; c < C; c += step) {
        const size_t at = base + c * a.inner;
        const A h = value(a, at);
        if (a.h) a.h[at] = (T)h;
        a.y[at] = (T)(weight(a, c) * (h * q));
    }
}

template <typename T, bool PLANES>
__global__ __launch_bounds__(256) void k_rms_backward(NormArgs<T> a) {
    typedef typename Acc<T>::type A;
    __shared__ A lds[256];
    const size_t tiles = PLANES ? (a.inner + 63) / 64 : 1;
    const size_t o = blockIdx.x / tiles, i = PLANES ? (blockIdx.x % tiles) * 64 + (threadIdx.x & 63) : 0;
    const int c0 = PLANES ? threadIdx.x >> 6 : threadIdx.x, step = PLANES ? 4 : 256;
    const int C = i < a.inner ? a.C : 0;
    const size_t base = o * a.C * a.inner + i;
    const A q = i < a.inner ? a.q[o * a.inner + i] : (A)0;
    A s = 0;
    for (int c = c0; c < C; c += step) {
        const size_t at = base + c * a.inner;
        s += weight(a, c) * (A)a.gy[at] * (value(a, at) * q);
    }
    if (!PLANES) s = sum_lanes(s);
    s = sum_waves<A>(s, lds) / (A)a.C;
    for (int c = c0; c < C; c += step) {
        const size_t at = base + c * a.inner;
        A d = q * (weight(a, c) * (A)a.gy[at] - value(a, at) * q * s);
        if (a.gh) d += (A)a.gh[at];
        a.dx[at] = (T)d;
    }
}

// partial[k][c] = sum of gy n over the k-th share of the pixels.  PLANES: one channel a workgroup; otherwise 256 channels a
// workgroup, a lane each.
template <typename T, bool PLANES>
__global__ __launch_bounds__(256) void k_rms_dw(NormArgs<T> a) {
    typedef typename Acc<T>::type A;
    __shared__ A lds[256];
    const size_t pixels = a.outer * a.inner;
    A s = 0;
    if (PLANES) {
        const int c = blockIdx.x;
        for (size_t p = (size_t)blockIdx.y * 256 + threadIdx.x; p < pixels; p += (size_t)gridDim.y * 256) {
            const size_t at = (p / a.inner * a.C + c) * a.inner + p % a.inner;
            s += (A)a.gy[at] * (value(a, at) * a.q[p]);
        }
        s = sum_waves<A>(sum_lanes(s), lds);
        if (threadIdx.x == 0) a.partial[(size_t)blockIdx.y * a.C + c] = s;
    } else {
        const int c = blockIdx.x * 256 + threadIdx.x;
        if (c >= a.C) return;
        for (size_t p = blockIdx.y; p < pixels; p += gridDim.y) s += (A)a.gy[p * a.C + c] * (value(a, p * a.C + c) * a.q[p]);
        a.partial[(size_t)blockIdx.y * a.C + c] = s;
    }
}

// dw[c] = sum of the partials, 64 channels a workgroup
template <typename T>
__global__ __launch_bounds__(256) void k_rms_dw_sum(NormArgs<T> a) {
    typedef typename Acc<T>::type A;
    __shared__ A lds[256];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63);
    A s = 0;
    if (c < a.C) for (int k = threadIdx.x >> 6; k < a.n_partial; k += 4) s += a.partial[(size_t)k * a.C + c];
    s = sum_waves<A>(s, lds);
    if (c < a.C && threadIdx.x < 64) {
        if (a.w32) static_cast<float*>(a.dw)[c] = (float)s;
        else static_cast<T*>(a.dw)[c] = (T)s;
    }
}

int partials(size_t pixels) { return (int)(pixels < 64 * 256 ? (pixels + 255) / 256 : 64); }

int launched(const char* who) {
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return ggs_fail_(GGS_ERR_HIP, "%s: launch failed: %s", who, hipGetErrorString(e));
    return GGS_OK;
}

template <typename T> int run_forward(NormArgs<T> a, hipStream_t s) {
    const size_t tiles = a.inner == 1 ? 1 : (a.inner + 63) / 64, blocks = a.outer * tiles;
    if (blocks > 0x7fffffffu) return ggs_fail_(GGS_ERR_SIZE, "ggs_rms_norm_forward: more than 2^31 workgroups");
    if (a.inner == 1) hipLaunchKernelGGL((k_rms_forward<T, false>), dim3((unsigned)blocks), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_rms_forward<T, true>), dim3((unsigned)blocks), dim3(256), 0, s, a);
    return launched("ggs_rms_norm_forward");
}

template <typename T> int run_backward(NormArgs<T> a, hipStream_t s) {
    const size_t tiles = a.inner == 1 ? 1 : (a.inner + 63) / 64, blocks = a.outer * tiles;
    if (blocks > 0x7fffffffu) return ggs_fail_(GGS_ERR_SIZE, "ggs_rms_norm_backward: more than 2^31 workgroups");
    if (a.inner == 1) hipLaunchKernelGGL((k_rms_backward<T, false>), dim3((unsigned)blocks), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_rms_backward<T, true>), dim3((unsigned)blocks), dim3(256), 0, s, a);
    int rc = launched("ggs_rms_norm_backward");
    if (rc != GGS_OK || !a.dw) return rc;
    a.n_partial = partials(a.outer * a.inner);
    if (a.inner == 1) hipLaunchKernelGGL((k_rms_dw<T, false>), dim3((a.C + 255) / 256, a.n_partial), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_rms_dw<T, true>), dim3(a.C, a.n_partial), dim3(256), 0, s, a);
    rc = launched("ggs_rms_norm_backward");
    if (rc != GGS_OK) return rc;
    hipLaunchKernelGGL((k_rms_dw_sum<T>), dim3((a.C + 63) / 64), dim3(256), 0, s, a);
    return launched("ggs_rms_norm_backward");
}

int check_sizes(const char* who, int dtype, size_t outer, int channels, size_t inner, double eps) {
    if (dtype < GGS_DTYPE_F32 || dtype > GGS_DTYPE_BF16) return ggs_fail_(GGS_ERR_ARG, "%s: dtype %d is not float / half / double / bfloat16", who, dtype);
    if (channels <= 0) return ggs_fail_(GGS_ERR_ARG, "%s: no channels", who);
    if (!(eps > 0.0)) return ggs_fail_(GGS_ERR_ARG, "%s: eps must be positive", who);
    if (inner && outer > ((size_t)1 << 46) / inner / (size_t)channels) return ggs_fail_(GGS_ERR_SIZE, "%s: more than 2^46 elements", who);
    return GGS_OK;
}

template <typename T>
NormArgs<T> norm_args(size_t outer, int channels, size_t inner, const void* x, const void* residual, const void* weight, int weight_f32, double eps) {
    NormArgs<T> a = {};
    a.outer = outer; a.inner = inner; a.C = channels;
    a.x = static_cast<const T*>(x); a.r = static_cast<const T*>(residual);
    a.w = weight; a.w32 = weight_f32 != 0; a.eps = (typename Acc<T>::type)eps;
    return a;
}

template <typename T>
int forward(size_t outer, int channels, size_t inner, const void* x, const void* residual, const void* weight, int weight_f32, double eps,
            void* y, void* h, void* q, hipStream_t s) {
    NormArgs<T> a = norm_args<T>(outer, channels, inner, x, residual, weight, weight_f32, eps);
    a.y = static_cast<T*>(y); a.h = static_cast<T*>(h); a.q = static_cast<typename Acc<T>::type*>(q);
    return run_forward(a, s);
}

template <typename T>
int backward(size_t outer, int channels, size_t inner, const void* x, const void* residual, const void* weight, int weight_f32, const void* q,
             const void* gy, const void* gh, void* dx, void* dw, void* workspace, hipStream_t s) {
    NormArgs<T> a = norm_args<T>(outer, channels, inner, x, residual, weight, weight_f32, 0.0);
    a.q = static_cast<typename Acc<T>::type*>(const_cast<void*>(q));
    a.gy = static_cast<const T*>(gy); a.gh = static_cast<const T*>(gh); a.dx = static_cast<T*>(dx);
    a.dw = dw; a.partial = static_cast<typename Acc<T>::type*>(workspace);
    return run_backward(a, s);
}

}  // namespace

extern "C" {

int ggs_rms_norm_forward(int dtype, size_t outer, int channels, size_t inner, const void* x, const void* residual,
                         const void* weight, int weight_f32, double eps, void* y, void* h, void* q, void* stream) {
    ggs_clear_error_();
    int rc = check_sizes("ggs_rms_norm_forward", dtype, outer, channels, inner, eps);
    if (rc != GGS_OK) return rc;
    if (outer == 0 || inner == 0) return GGS_OK;
    if (!x || !y) return ggs_fail_(GGS_ERR_ARG, "ggs_rms_norm_forward: NULL pointer argument");
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case GGS_DTYPE_F32: return forward<float>(outer, channels, inner, x, residual, weight, weight_f32, eps, y, h, q, s);
        case GGS_DTYPE_F16: return forward<_Float16>(outer, channels, inner, x, residual, weight, weight_f32, eps, y, h, q, s);
        case GGS_DTYPE_BF16: return forward<__bf16>(outer, channels, inner, x, residual, weight, weight_f32, eps, y, h, q, s);
        default: return forward<double>(outer, channels, inner, x, residual, weight, weight_f32, eps, y, h, q, s);
    }
}

size_t ggs_rms_norm_workspace_bytes(int dtype, size_t outer, int channels, size_t inner) {
    if (channels <= 0 || outer == 0 || inner == 0) return 0;
    return (size_t)partials(outer * inner) * (size_t)channels * (dtype == GGS_DTYPE_F64 ? 8 : 4);
}

int ggs_rms_norm_backward(int dtype, size_t outer, int channels, size_t inner, const void* x, const void* residual,
                          const void* weight, int weight_f32, const void* q, const void* gy, const void* gh, void* dx,
                          void* dw, void* workspace, size_t workspace_bytes, void* stream) {
    ggs_clear_error_();
    int rc = check_sizes("ggs_rms_norm_backward", dtype, outer, channels, inner, 1.0);
    if (rc != GGS_OK) return rc;
    if (outer == 0 || inner == 0) return GGS_OK;
    if (!x || !q || !gy || !dx) return ggs_fail_(GGS_ERR_ARG, "ggs_rms_norm_backward: NULL pointer argument");
    if (dw && (!workspace || workspace_bytes < ggs_rms_norm_workspace_bytes(dtype, outer, channels, inner)))
        return ggs_fail_(GGS_ERR_SIZE, "ggs_rms_norm_backward: the workspace is too small (ggs_rms_norm_workspace_bytes)");
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case GGS_DTYPE_F32: return backward<float>(outer, channels, inner, x, residual, weight, weight_f32, q, gy, gh, dx, dw, workspace, s);
        case GGS_DTYPE_F16: return backward<_Float16>(outer, channels, inner, x, residual, weight, weight_f32, q, gy, gh, dx, dw, workspace, s);
        case GGS_DTYPE_BF16: return backward<__bf16>(outer, channels, inner, x, residual, weight, weight_f32, q, gy, gh, dx, dw, workspace, s);
        default: return backward<double>(outer, channels, inner, x, residual, weight, weight_f32, q, gy, gh, dx, dw, workspace, s);
    }
}

}  // extern "C"
