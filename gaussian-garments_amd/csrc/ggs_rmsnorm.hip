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
// The backward pass of the backward pass, from the cotangents v of dx and u_c of dw_c, with the means over the channels
// s = mean(w gy n), b = mean(v n), m = mean(v w gy), t = mean(u gy n):
//   to gy: w q (v - n b) + u n,   to w: sum over pixels of q gy (v - n b),   to gh: v,
//   to h:  q^2 (n (3 s b - m) - b w gy - s v) - q n t + q u gy
// HBM-bound: forward reads x, r and writes y, h; backward reads h (x, r), gy, gh and writes dx: at most 4 and 5 elements a value.
// Measured (replayed from a graph, inputs of three passes in turn; a copy of 2 GiB runs at 4.9 TB/s here):
//   2 x 128 x 256 x 256 float     forward 51.5 us (5.2 TB/s), backward 52.6 us (5.1 TB/s)
//   512 x 64 x 64 float                    7.7 us (4.3),                11.3 us (3.7)      64 ... 256 workgroups: one round of loads
//   32 x 1024 x 1024 half                 57.7 us (4.7)
//   100000 x 51 float, no residual         8.8 us (4.7),                16.0 us (3.8)      3 us of it the sum of the dw partials
//   4096 x 4096 bf16                      21.0 us (6.4, part of it from the caches), 40.8 us (4.1)
//   3 x 100 x 37 x 53 half                 5.7 us,                       8.6 us            launches
#include "ggs_kernels.h"

namespace {

template <typename T> struct Acc { typedef float type; };
template <> struct Acc<double> { typedef double type; };

template <typename T> struct NormArgs {
    typedef typename Acc<T>::type A;
    size_t outer, inner;
    int C;
    const T *x, *r, *gy, *gh, *v;
    const void *w, *u;
    bool w32;                    // w, u (and dw) are float whatever T is
    A eps, inv_c;                // 1 / C
    T *y, *h, *dx, *dgy;
    A *q, *b;                    // [outer][inner]
    A* partial;                  // [n_partial][C]
    int n_partial;
    void* dw;
};

template <typename T> __device__ __forceinline__ typename Acc<T>::type per_channel(const NormArgs<T>& a, const void* w, int c, int absent) {
    typedef typename Acc<T>::type A;
    if (!w) return (A)absent;
    return a.w32 ? (A) static_cast<const float*>(w)[c] : (A) static_cast<const T*>(w)[c];
}
template <typename T> __device__ __forceinline__ typename Acc<T>::type weight(const NormArgs<T>& a, int c) { return per_channel(a, a.w, c, 1); }
template <typename T> __device__ __forceinline__ typename Acc<T>::type value(const NormArgs<T>& a, size_t at) {
    typedef typename Acc<T>::type A;
    return a.r ? (A)a.x[at] + (A)a.r[at] : (A)a.x[at];
}

// Sum over the W waves of a workgroup, lane by lane.
template <int W, typename A> __device__ __forceinline__ A sum_waves(A s, A* lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __syncthreads();
    lds[wave * 64 + lane] = s;
    __syncthreads();
    s = 0;
#pragma unroll
    for (int k = 0; k < W; ++k) s += lds[k * 64 + lane];
    return s;
}
template <typename A> __device__ __forceinline__ A sum_lanes(A s) {
#pragma unroll
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
    return s;
}

// Any channel count, two passes over the data (the second one from the caches).  PLANES: 64 pixels of one map at a time, the
// workgroup's sixteen waves take every sixteenth channel; otherwise one row at a time.  Element-wide accesses, so 2 x 1100 x
// 64 x 64 float takes 67.7 us forward and 94.8 us backward (2.1 and 1.5 TB/s): 128 tiles on 256 CUs.
template <typename T, bool PLANES>
__global__ __launch_bounds__(1024) void k_rms_forward(NormArgs<T> a) {
    typedef typename Acc<T>::type A;
    __shared__ A lds[1024];
    const size_t tiles = PLANES ? (a.inner + 63) / 64 : 1;
    const int c0 = PLANES ? threadIdx.x >> 6 : threadIdx.x, step = PLANES ? 16 : 1024;
    for (size_t tile = blockIdx.x; tile < a.outer * tiles; tile += gridDim.x) {
        const size_t o = tile / tiles, i = PLANES ? (tile % tiles) * 64 + (threadIdx.x & 63) : 0;
        const int C = i < a.inner ? a.C : 0;                        // lanes beyond the map only take part in the barriers
        const size_t base = o * a.C * a.inner + i;
        A s = 0;
        for (int c = c0; c < C; c += step) {
            const A h = value(a, base + c * a.inner);
            s += h * h;
        }
        if (!PLANES) s = sum_lanes(s);
        s = sum_waves<16>(s, lds);
        const A q = (A)1 / sqrt(s / (A)a.C + a.eps);
        if (c0 == 0 && a.q && i < a.inner) a.q[o * a.inner + i] = q;
        for (int c = c0; c < C; c += step) {
            const size_t at = base + c * a.inner;
            const A h = value(a, at);
            if (a.h) a.h[at] = (T)h;
            a.y[at] = (T)(weight(a, c) * (h * q));
        }
    }
}

template <typename T, bool PLANES>
__global__ __launch_bounds__(1024) void k_rms_backward(NormArgs<T> a) {
    typedef typename Acc<T>::type A;
    __shared__ A lds[1024];
    const size_t tiles = PLANES ? (a.inner + 63) / 64 : 1;
    const int c0 = PLANES ? threadIdx.x >> 6 : threadIdx.x, step = PLANES ? 16 : 1024;
    for (size_t tile = blockIdx.x; tile < a.outer * tiles; tile += gridDim.x) {
        const size_t o = tile / tiles, i = PLANES ? (tile % tiles) * 64 + (threadIdx.x & 63) : 0;
        const int C = i < a.inner ? a.C : 0;
        const size_t base = o * a.C * a.inner + i;
        const A q = i < a.inner ? a.q[o * a.inner + i] : (A)0;
        A s = 0;
        for (int c = c0; c < C; c += step) {
            const size_t at = base + c * a.inner;
            s += weight(a, c) * (A)a.gy[at] * (value(a, at) * q);
        }
        if (!PLANES) s = sum_lanes(s);
        s = sum_waves<16>(s, lds) / (A)a.C;
        for (int c = c0; c < C; c += step) {
            const size_t at = base + c * a.inner;
            A d = q * (weight(a, c) * (A)a.gy[at] - value(a, at) * q * s);
            if (a.gh) d += (A)a.gh[at];
            a.dx[at] = (T)d;
        }
    }
}

// The backward pass of the backward pass, in the shape of the two kernels above: four sums, then the gradients to h and gy, and
// b for k_rms_dw.  No training loop here takes second derivatives every step: kept simple (2 x 128 x 256 x 256 float: 129 us with
// the sums over the pixels, bound by its two passes and element-wide accesses).
template <typename T, bool PLANES>
__global__ __launch_bounds__(1024) void k_rms_second(NormArgs<T> a) {
    typedef typename Acc<T>::type A;
    __shared__ A lds[1024];
    const size_t tiles = PLANES ? (a.inner + 63) / 64 : 1;
    const int c0 = PLANES ? threadIdx.x >> 6 : threadIdx.x, step = PLANES ? 16 : 1024;
    for (size_t tile = blockIdx.x; tile < a.outer * tiles; tile += gridDim.x) {
        const size_t o = tile / tiles, i = PLANES ? (tile % tiles) * 64 + (threadIdx.x & 63) : 0;
        const int C = i < a.inner ? a.C : 0;
        const size_t base = o * a.C * a.inner + i;
        const A q = i < a.inner ? a.q[o * a.inner + i] : (A)0;
        A sum[4] = {};                                              // s, b, m, t
        for (int c = c0; c < C; c += step) {
            const size_t at = base + c * a.inner;
            const A n = value(a, at) * q, g = (A)a.gy[at], w = weight(a, c) * g, v = a.v ? (A)a.v[at] : (A)0;
            sum[0] += w * n; sum[1] += v * n; sum[2] += v * w; sum[3] += per_channel(a, a.u, c, 0) * g * n;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (!PLANES) sum[k] = sum_lanes(sum[k]);
            sum[k] = sum_waves<16>(sum[k], lds) / (A)a.C;
        }
        if (c0 == 0 && i < a.inner) a.b[o * a.inner + i] = sum[1];
        for (int c = c0; c < C; c += step) {
            const size_t at = base + c * a.inner;
            const A n = value(a, at) * q, g = (A)a.gy[at], w = weight(a, c), v = a.v ? (A)a.v[at] : (A)0, u = per_channel(a, a.u, c, 0);
            a.dx[at] = (T)(q * (q * (n * ((A)3 * sum[0] * sum[1] - sum[2]) - sum[1] * (w * g) - sum[0] * v) - n * sum[3] + u * g));
            a.dgy[at] = (T)(w * q * (v - n * sum[1]) + u * n);
        }
    }
}

// partial[k][c] = sum over the k-th share of the pixels of gy n (SECOND: of q gy (v - n b)).  PLANES: one channel a workgroup;
// otherwise 256 channels a workgroup, a lane each.
template <typename T, bool SECOND> __device__ __forceinline__ typename Acc<T>::type dw_term(const NormArgs<T>& a, size_t at, size_t p) {
    typedef typename Acc<T>::type A;
    const A n = value(a, at) * a.q[p], g = (A)a.gy[at];
    return SECOND ? a.q[p] * g * ((a.v ? (A)a.v[at] : (A)0) - n * a.b[p]) : g * n;
}
template <typename T, bool PLANES, bool SECOND>
__global__ __launch_bounds__(256) void k_rms_dw(NormArgs<T> a) {
    typedef typename Acc<T>::type A;
    __shared__ A lds[256];
    const size_t pixels = a.outer * a.inner;
    A s = 0;
    if (PLANES) {
        const int c = blockIdx.x;
        for (size_t p = (size_t)blockIdx.y * 256 + threadIdx.x; p < pixels; p += (size_t)gridDim.y * 256)
            s += dw_term<T, SECOND>(a, (p / a.inner * a.C + c) * a.inner + p % a.inner, p);
        s = sum_waves<4>(sum_lanes(s), lds);
        if (threadIdx.x == 0) a.partial[(size_t)blockIdx.y * a.C + c] = s;
    } else {
        const int c = blockIdx.x * 256 + threadIdx.x;
        if (c >= a.C) return;
        for (size_t p = blockIdx.y; p < pixels; p += gridDim.y) s += dw_term<T, SECOND>(a, p * a.C + c, p);
        a.partial[(size_t)blockIdx.y * a.C + c] = s;
    }
}

// dw[c] = sum of the partials, 8 channels a workgroup, 128 rows of partials at a time (2 - 4 us: a launch and one round of loads)
template <typename T>
__global__ __launch_bounds__(1024) void k_rms_dw_sum(NormArgs<T> a) {
    typedef typename Acc<T>::type A;
    __shared__ A lds[16][8];
    const int lc = threadIdx.x & 7, row = threadIdx.x >> 3, c = blockIdx.x * 8 + lc;
    A s = 0;
    if (c < a.C) for (int k = row; k < a.n_partial; k += 128) s += a.partial[(size_t)k * a.C + c];
#pragma unroll
    for (int d = 8; d < 64; d <<= 1) s += __shfl_xor(s, d);
    if ((threadIdx.x & 63) < 8) lds[threadIdx.x >> 6][lc] = s;
    __syncthreads();
    if (row) return;
    s = 0;
#pragma unroll
    for (int k = 0; k < 16; ++k) s += lds[k][lc];
    if (c < a.C) {
        if (a.w32) static_cast<float*>(a.dw)[c] = (float)s;
        else static_cast<T*>(a.dw)[c] = (T)s;
    }
}

// ---- one pass over the data: a pixel's channels stay in registers ----------------------------------------------------------
// VEC elements at any element address as one access (unaligned accesses are legal on this part).  Addresses are a base that is
// the same for the whole workgroup plus 32-bit byte offsets a lane, which all tensors of a pixel share.
template <typename T, int VEC> struct __attribute__((packed, aligned(alignof(T)))) Pack { T v[VEC]; };
typedef unsigned Bits16 __attribute__((ext_vector_type(4), aligned(2)));
// NT: past the caches (see STREAM_BYTES)
template <typename T, int VEC, bool NT = false> __device__ __forceinline__ Pack<T, VEC> fetch(const T* base, unsigned off) {
    const char* at = reinterpret_cast<const char*>(base) + off;
    if constexpr (sizeof(Pack<T, VEC>) == 16) {
        const Bits16* p = reinterpret_cast<const Bits16*>(at);
        const Bits16 v = NT ? __builtin_nontemporal_load(p) : *p;
        Pack<T, VEC> o;
        __builtin_memcpy(&o, &v, 16);
        return o;
    } else {
        return *reinterpret_cast<const Pack<T, VEC>*>(at);
    }
}
// A pack that stays in registers between phases: as four words, where the compiler would give every 16-bit element one
template <typename T, int VEC, bool WIDE = sizeof(T) * VEC == 16> struct Kept {
    Bits16 b;
    // an unpacked copy does not outlive this point
    __device__ __forceinline__ void pin() { asm volatile("" : "+v"(b[0]), "+v"(b[1]), "+v"(b[2]), "+v"(b[3])); }
    __device__ __forceinline__ void operator=(const Pack<T, VEC>& p) { __builtin_memcpy(&b, &p, 16); }
    __device__ __forceinline__ Pack<T, VEC> get() const { Pack<T, VEC> p; __builtin_memcpy(&p, &b, 16); return p; }
};
template <typename T, int VEC> struct Kept<T, VEC, false> {
    Pack<T, VEC> p;
    __device__ __forceinline__ void pin() {}
    __device__ __forceinline__ void operator=(const Pack<T, VEC>& o) { p = o; }
    __device__ __forceinline__ Pack<T, VEC> get() const { return p; }
};
// Whole 16-byte vectors are stored past the caches: what they would push out are the inputs that other workgroups are about to
// read (4096 x 4096 bf16 forward 29.3 -> 22.0 us, 256 x 128 x 128 float backward 16.8 -> 15.5 us).
template <typename T, int VEC> __device__ __forceinline__ void put(T* base, unsigned off, const float (&v)[VEC]) {
    Pack<T, VEC> o;
#pragma unroll
    for (int j = 0; j < VEC; ++j) o.v[j] = (T)v[j];
    char* at = reinterpret_cast<char*>(base) + off;
    if constexpr (sizeof(o) == 16) {
        Bits16 b;
        __builtin_memcpy(&b, &o, 16);
        __builtin_nontemporal_store(b, reinterpret_cast<Bits16*>(at));
    } else {
        *reinterpret_cast<Pack<T, VEC>*>(at) = o;
    }
}
// The vectors of one tensor for the K channels of a thread, all on their way before the first is needed (a branch or a
// conversion in between would wait for each); zeros for a tensor that is not there.
template <typename T, int VEC, int K, bool NT = false>
__device__ __forceinline__ void fetch_all(const T* base, const unsigned (&off)[K], Kept<T, VEC> (&v)[K]) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = fetch<T, VEC, NT>(base, off[k]);
}
template <typename T, int VEC, int K, bool NT = false>
__device__ __forceinline__ void fetch_some(const T* t, size_t base, const unsigned (&off)[K], Kept<T, VEC> (&v)[K]) {
    if (t) fetch_all<T, VEC, K, NT>(t + base, off, v);
    else {
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = Pack<T, VEC>{};
    }
}
template <typename T, int VEC, int K>
__device__ __forceinline__ void add_up(const Kept<T, VEC> (&x)[K], const Kept<T, VEC> (&r)[K], float (&h)[K][VEC]) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const Pack<T, VEC> a = x[k].get(), b = r[k].get();
#pragma unroll
        for (int j = 0; j < VEC; ++j) h[k][j] = (float)a.v[j] + (float)b.v[j];
    }
}

// Channels-first maps.  Registers and not LDS hold the tile: 64 pixels of 512 float channels are 128 KB, a quarter of a CU's
// registers and most of its LDS, and the sums need only one value a pixel exchanged.  A workgroup takes LP VEC neighbouring
// pixels of one map and all their channels: LP lanes of a wave lie along the pixels, its other 64 / LP lanes and the waves along
// the channels, K channels a thread.  The last tile of a map is moved back to end with the map: pixels that two tiles hold get
// the same values from both, and count once in dw.
template <int VEC, int LP> struct PlaneTile {
    static constexpr int LC = 64 / LP, TP = LP * VEC;
    int c0, step;                            // first channel of this thread, channel step
    size_t base, q_base;                     // of the map
    unsigned i0;                             // first pixel of this lane's vector
    int fresh;                               // its first pixel that no vector before holds
    template <typename T> __device__ __forceinline__ PlaneTile(const NormArgs<T>& a, unsigned tile) {
        const unsigned tiles = ((unsigned)a.inner + TP - 1) / TP, o = tile / tiles;
        const int lane = threadIdx.x & 63;
        const unsigned i = (tile - o * tiles) * TP + (lane % LP) * VEC, last = (unsigned)a.inner - VEC;
        i0 = i < last ? i : last;
        fresh = (int)(i - i0 < (unsigned)VEC ? i - i0 : VEC);
        c0 = (threadIdx.x >> 6) * LC + lane / LP;
        step = (blockDim.x >> 6) * LC;
        base = (size_t)o * a.C * a.inner;
        q_base = (size_t)o * a.inner;
    }
    // Byte offsets of this thread's channels within the map; a channel beyond the last one reads the last one.
    template <typename T, int K> __device__ __forceinline__ void offsets(const NormArgs<T>& a, unsigned (&off)[K]) const {
#pragma unroll
        for (int k = 0; k < K; ++k) off[k] = ((unsigned)min(c0 + k * step, a.C - 1) * (unsigned)a.inner + i0) * (unsigned)sizeof(T);
    }
    // Their weights, the same for every tile.
    template <typename T, int K> static __device__ __forceinline__ void weights(const NormArgs<T>& a, float (&w)[K]) {
        const unsigned c0 = (threadIdx.x >> 6) * LC + (threadIdx.x & 63) / LP, step = (blockDim.x >> 6) * LC, last = a.C - 1;
#pragma unroll
        for (int k = 0; k < K; ++k) w[k] = 1.0f;
        if (a.w && a.w32) {
#pragma unroll
            for (int k = 0; k < K; ++k) w[k] = static_cast<const float*>(a.w)[min(c0 + k * step, last)];
        } else if (a.w) {
#pragma unroll
            for (int k = 0; k < K; ++k) w[k] = (float)static_cast<const T*>(a.w)[min(c0 + k * step, last)];
        }
    }
};

// Sums over the lanes of a wave that hold the same pixels, then over the waves.
template <int VEC, int LP> __device__ __forceinline__ void sum_channels(float (&s)[VEC], float* lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
    for (int d = LP; d < 64; d <<= 1) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) s[j] += __shfl_xor(s[j], d);
    }
    if (waves == 1) return;
    if (lane < LP) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) lds[(wave * LP + lane) * VEC + j] = s[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < VEC; ++j) s[j] = 0.0f;
#pragma unroll 2
    for (int k = 0; k < waves; ++k) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) s[j] += lds[(k * LP + lane % LP) * VEC + j];
    }
}

template <typename T, int VEC, int LP, int K, bool NT>
__global__ __launch_bounds__(1024) void k_planes_forward(NormArgs<T> a) {
    __shared__ float lds[16 * LP * VEC];
    const PlaneTile<VEC, LP> t(a, blockIdx.x);
    unsigned off[K];
    Kept<T, VEC> x[K], r[K];
    float h[K][VEC], w[K], s[VEC] = {};
    t.offsets(a, off);
    fetch_all<T, VEC, K, NT>(a.x + t.base, off, x);
    fetch_some<T, VEC, K, NT>(a.r, t.base, off, r);
    t.weights(a, w);
    add_up<T, VEC, K>(x, r, h);
#pragma unroll
    for (int k = 0; k < K; ++k) if (t.c0 + k * t.step < a.C) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) s[j] = fmaf(h[k][j], h[k][j], s[j]);
    }
    sum_channels<VEC, LP>(s, lds);
#pragma unroll
    for (int j = 0; j < VEC; ++j) s[j] = rsqrtf(s[j] * a.inv_c + a.eps);
    if (t.c0 == 0 && a.q) put<float, VEC>(a.q + t.q_base, t.i0 * 4u, s);
#pragma unroll
    for (int k = 0; k < K; ++k) if (t.c0 + k * t.step < a.C) {
        float y[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) y[j] = w[k] * (h[k][j] * s[j]);
        if (a.h) put<T, VEC>(a.h + t.base, off[k], h[k]);
        put<T, VEC>(a.y + t.base, off[k], y);
    }
}

// A workgroup walks tiles with a fixed stride and keeps its share of dw in registers meanwhile: one row of partials each.  (Its own
// reduction a tile would cost as many shuffles as there are channels.)
template <typename T, int VEC, int LP, int K, bool NT>
__global__ __launch_bounds__(1024) void k_planes_backward(NormArgs<T> a, unsigned tiles) {
    __shared__ float lds[2][16 * LP * VEC];
    // gh on its way with the rest, or after the sums where its registers are not there.  (16 bits with four channels a thread, the
    // blocks of 257 - 1024 channels, spill 3 - 5 of 128 registers even so: 2 x 512 x 128 x 128 bf16 44 us, 34 at the copy rate.)
    constexpr bool EARLY = K * VEC <= 16;
    float dw[K] = {}, w[K];
    int turn = 0;
    PlaneTile<VEC, LP>::weights(a, w);
    for (unsigned tile = blockIdx.x; tile < tiles; tile += gridDim.x, turn ^= 1) {
        const PlaneTile<VEC, LP> t(a, tile);
        unsigned off[K];
        Kept<T, VEC> x[K], r[K], g[K], gh[K];
        float h[K][VEC], s[VEC] = {};
        t.offsets(a, off);
        fetch_all<T, VEC, K, NT>(a.x + t.base, off, x);
        fetch_some<T, VEC, K, NT>(a.r, t.base, off, r);
        fetch_all<T, VEC, K, NT>(a.gy + t.base, off, g);
        const Pack<float, VEC> q = fetch<float, VEC>(a.q + t.q_base, t.i0 * 4u);
        if (EARLY) fetch_some<T, VEC, K, NT>(a.gh, t.base, off, gh);
        add_up<T, VEC, K>(x, r, h);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const Pack<T, VEC> gy = g[k].get();
#pragma unroll
            for (int j = 0; j < VEC; ++j) h[k][j] *= q.v[j];
            if (t.c0 + k * t.step < a.C) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float gn = (float)gy.v[j] * h[k][j];
                    dw[k] += j >= t.fresh ? gn : 0.0f;
                    s[j] = fmaf(w[k], gn, s[j]);
                }
            }
        }
        sum_channels<VEC, LP>(s, lds[turn]);
        if (!EARLY) {
            fetch_some<T, VEC, K, NT>(a.gh, t.base, off, gh);
#pragma unroll
            for (int k = 0; k < K; ++k) g[k].pin();
        }
#pragma unroll
        for (int k = 0; k < K; ++k) if (t.c0 + k * t.step < a.C) {
            const Pack<T, VEC> gy = g[k].get(), more = gh[k].get();
            float d[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) d[j] = fmaf(q.v[j], (float)gy.v[j] * w[k] - h[k][j] * (s[j] * a.inv_c), (float)more.v[j]);
            put<T, VEC>(a.dx + t.base, off[k], d);
        }
    }
    if (!a.dw) return;
    constexpr int LC = 64 / LP;
    const int lane = threadIdx.x & 63, c0 = (threadIdx.x >> 6) * LC + lane / LP, step = (blockDim.x >> 6) * LC;
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int d = 1; d < LP; d <<= 1) dw[k] += __shfl_xor(dw[k], d);
        if (lane % LP == 0 && c0 + k * step < a.C) a.partial[(size_t)blockIdx.x * a.C + c0 + k * step] = dw[k];
    }
}

// Rows of contiguous channels: G lanes a row, K vectors of VEC channels a lane.  The last vector of a row is moved back to end
// with the row: channels that two vectors hold count once in the sums.
template <int VEC, int G> struct RowSlot {
    int lane;                                // within the row's lanes
    __device__ __forceinline__ RowSlot() : lane(threadIdx.x % G) {}
    __device__ __forceinline__ bool on(int k, int C) const { return (lane + k * G) * VEC < C; }
    __device__ __forceinline__ int at(int k, int C) const { const int c = (lane + k * G) * VEC; return c < C - VEC ? c : C - VEC; }
    __device__ __forceinline__ int fresh(int k, int C) const { return (lane + k * G) * VEC - at(k, C); }
};

// Sum over the G lanes of a row (rows of more than a wave: G / 64 waves, `lds` one float a wave of the workgroup).
template <int G> __device__ __forceinline__ float sum_row(float s, float* lds) {
#pragma unroll
    for (int d = 1; d < (G < 64 ? G : 64); d <<= 1) s += __shfl_xor(s, d);
    if (G > 64) {
        const int wave = threadIdx.x >> 6, first = wave / (G / 64) * (G / 64);
        if ((threadIdx.x & 63) == 0) lds[wave] = s;
        __syncthreads();
        s = 0.0f;
#pragma unroll
        for (int k = 0; k < G / 64; ++k) s += lds[first + k];
    }
    return s;
}

template <typename T, int VEC, int G, int K>
__device__ __forceinline__ void row_weights(const NormArgs<T>& a, const RowSlot<VEC, G>& t, float (&w)[K][VEC]) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) w[k][j] = 1.0f;
    }
    if (a.w && a.w32) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const Pack<float, VEC> p = fetch<float, VEC>(static_cast<const float*>(a.w), t.at(k, a.C) * 4u);
#pragma unroll
            for (int j = 0; j < VEC; ++j) w[k][j] = p.v[j];
        }
    } else if (a.w) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const Pack<T, VEC> p = fetch<T, VEC>(static_cast<const T*>(a.w), t.at(k, a.C) * (unsigned)sizeof(T));
#pragma unroll
            for (int j = 0; j < VEC; ++j) w[k][j] = (float)p.v[j];
        }
    }
}

template <typename T, int VEC, int G, int K>
__global__ __launch_bounds__(G > 256 ? G : 256) void k_rows_forward(NormArgs<T> a) {
    constexpr int THREADS = G > 256 ? G : 256, ROWS = THREADS / G;
    __shared__ float lds[16];
    const RowSlot<VEC, G> t;
    const size_t row0 = (size_t)blockIdx.x * ROWS, base = row0 * a.C;
    const unsigned rows = (unsigned)min((size_t)ROWS, a.outer - row0), mine = threadIdx.x / G, row = min(mine, rows - 1);
    unsigned off[K];
    Kept<T, VEC> x[K], r[K];
    float h[K][VEC], w[K][VEC], s = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) off[k] = (row * a.C + t.at(k, a.C)) * (unsigned)sizeof(T);
    fetch_all<T, VEC, K>(a.x + base, off, x);
    fetch_some<T, VEC, K>(a.r, base, off, r);
    row_weights(a, t, w);
    add_up<T, VEC, K>(x, r, h);
#pragma unroll
    for (int k = 0; k < K; ++k) if (t.on(k, a.C)) {
        const int fresh = t.fresh(k, a.C);
#pragma unroll
        for (int j = 0; j < VEC; ++j) s = j >= fresh ? fmaf(h[k][j], h[k][j], s) : s;
    }
    s = sum_row<G>(s, lds);
    const float q = rsqrtf(s * a.inv_c + a.eps);
    if (mine >= rows) return;
    if (t.lane == 0 && a.q) a.q[row0 + row] = q;
#pragma unroll
    for (int k = 0; k < K; ++k) if (t.on(k, a.C)) {
        float y[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) y[j] = w[k][j] * (h[k][j] * q);
        if (a.h) put<T, VEC>(a.h + base, off[k], h[k]);
        put<T, VEC>(a.y + base, off[k], y);
    }
}

// A workgroup of 1024 threads walks sets of 1024 / G rows and keeps its share of dw in registers meanwhile.
template <typename T, int VEC, int G, int K>
__global__ __launch_bounds__(1024) void k_rows_backward(NormArgs<T> a, unsigned sets) {
    constexpr int ROWS = 1024 / G;
    constexpr bool EARLY = K * VEC <= 16 && K < 4;       // gh: as in k_planes_backward
    __shared__ float lds[2][16], sum[G * K * VEC];
    const RowSlot<VEC, G> t;
    const unsigned mine = threadIdx.x / G;
    float dw[K][VEC] = {}, w[K][VEC];
    int turn = 0;
    row_weights(a, t, w);
    for (unsigned set = blockIdx.x; set < sets; set += gridDim.x, turn ^= 1) {
        const size_t row0 = (size_t)set * ROWS, base = row0 * a.C;
        const unsigned rows = (unsigned)min((size_t)ROWS, a.outer - row0), row = min(mine, rows - 1);
        const bool in = mine < rows;
        unsigned off[K];
        Kept<T, VEC> x[K], r[K], g[K], gh[K];
        float h[K][VEC], s = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) off[k] = (row * a.C + t.at(k, a.C)) * (unsigned)sizeof(T);
        fetch_all<T, VEC, K>(a.x + base, off, x);
        fetch_some<T, VEC, K>(a.r, base, off, r);
        fetch_all<T, VEC, K>(a.gy + base, off, g);
        const float q = a.q[row0 + row];
        if (EARLY) fetch_some<T, VEC, K>(a.gh, base, off, gh);
        add_up<T, VEC, K>(x, r, h);
#pragma unroll
        for (int k = 0; k < K; ++k) if (in && t.on(k, a.C)) {
            const int fresh = t.fresh(k, a.C);
            const Pack<T, VEC> gy = g[k].get();
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                h[k][j] *= q;
                const float gn = (float)gy.v[j] * h[k][j];
                dw[k][j] += gn;
                s = j >= fresh ? fmaf(w[k][j], gn, s) : s;
            }
        }
        s = sum_row<G>(s, lds[turn]) * a.inv_c;
        if (!EARLY) {
            fetch_some<T, VEC, K>(a.gh, base, off, gh);
#pragma unroll
            for (int k = 0; k < K; ++k) g[k].pin();
        }
#pragma unroll
        for (int k = 0; k < K; ++k) if (in && t.on(k, a.C)) {
            const Pack<T, VEC> gy = g[k].get(), more = gh[k].get();
            float d[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) d[j] = fmaf(q, (float)gy.v[j] * w[k][j] - h[k][j] * s, (float)more.v[j]);
            put<T, VEC>(a.dx + base, off[k], d);
        }
    }
    if (!a.dw) return;
    // the rows of one wave by shuffles, then the waves one after the other in LDS (a fixed order)
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
#pragma unroll
            for (int d = G; d < 64; d <<= 1) dw[k][j] += __shfl_xor(dw[k][j], d);
        }
    }
    constexpr int TURNS = G < 64 ? 16 : ROWS;
    const int my_turn = G < 64 ? threadIdx.x >> 6 : threadIdx.x / G;
    const bool first = G >= 64 || (threadIdx.x & 63) < G;
    for (int r = 0; r < TURNS; ++r) {
        if (r == my_turn && first) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    float* at = sum + (k * G + t.lane) * VEC + j;
                    *at = r ? *at + dw[k][j] : dw[k][j];
                }
            }
        }
        __syncthreads();
    }
    // vector v holds channels v VEC ... but the last one, which ends with the row
    const int vecs = (a.C + VEC - 1) / VEC;
    for (int c = threadIdx.x; c < a.C; c += 1024) {
        const int v = c / VEC, j = v == vecs - 1 ? c - (a.C - VEC) : c % VEC;
        a.partial[(size_t)blockIdx.x * a.C + c] = sum[v * VEC + j];
    }
}

// ---- which kernel ----------------------------------------------------------------------------------------------------------
// One-pass kernels: float and 16-bit types, a pixel's channels within the registers of one workgroup (1024 channels of a map,
// 16384 of a row), a map and its q within 32-bit offsets; the two-pass kernels serve double and what is left.
struct Plan {
    int kind;                    // 0 two passes, 1 planes, 2 rows
    int vec, lanes, k, waves;    // planes: LP and waves of a workgroup; rows: G
    size_t tiles;                // planes: tiles of all maps; rows: sets of 1024 / G rows
    int partials;
};

// Shares of the pixels in k_rms_dw: 256 pixels each and at most 64 for maps, 16 each and at most 256 for rows.
int two_pass_partials(size_t outer, size_t inner) {
    const size_t each = inner == 1 ? 16 : 256, most = inner == 1 ? 256 : 64, n = (outer * inner + each - 1) / each;
    return (int)(n < most ? n : most);
}

template <typename T> Plan plan(size_t outer, int C, size_t inner) {
    Plan p = {};
    constexpr int FULL = 16 / sizeof(T);
    const size_t pixels = outer * inner;
    p.partials = two_pass_partials(outer, inner);
    if (sizeof(T) == 8) return p;
    if (inner == 1) {
        const int vec = C >= FULL ? FULL : 1, vecs = (C + vec - 1) / vec;
        const int lanes = vecs <= 8 ? 4 : vecs <= 32 ? 16 : vecs <= 128 ? 64 : vecs <= 512 ? 256 : 1024;
        const size_t sets = (outer + 1024 / lanes - 1) / (1024 / lanes);
        if (vecs > (sizeof(T) == 4 ? 4096 : 2048) || sets > 0x7fffffffu) return p;
        p.kind = 2; p.vec = vec; p.lanes = lanes; p.k = vecs <= lanes ? 1 : vecs <= 2 * lanes ? 2 : 4; p.tiles = sets;
        p.partials = (int)(sets < 256 ? sets : 256);          // (128 / 256 / 512: 4096 x 4096 bf16 backward 58.6 / 45.3 / 47.1 us)
        return p;
    }
    // (the 32-bit byte offsets are those of a map of T and of its q, float whatever T is: one channel in 16 bits is the case where
    // the second bound is the smaller one)
    if (C > 1024 || (size_t)C * inner > 0xffffffffu / sizeof(T) || inner > 0xffffffffu / sizeof(float)) return p;
    p.vec = inner >= (size_t)FULL ? FULL : 1;
    // Lanes along the pixels: 16 (float) or 8 make 256 / 128 bytes of every channel, 4 make 64 and more workgroups.  Forward us of
    // 256 float channels with 4 / 8 / 16 lanes: 32 x 32 pixels 3.9 / 4.2 / 5.2, 64 x 64 6.8 / 5.5 / 6.5, 128 x 128 17.8 / 12.5 /
    // 12.8; 2 x 128 x 256 x 256 82 / 58 / 55.
    p.lanes = p.vec == 1 || pixels < 2048 ? 4 : pixels < 32768 ? 8 : 64 / FULL;
    while (C > 64 * 64 / p.lanes) p.lanes /= 2;                // 16 waves of 64 / lanes channels, 4 a thread
    const int units = (C + 64 / p.lanes - 1) / (64 / p.lanes);
    // As many waves as there may be before a thread takes more channels (2 x 128 x 256 x 256 float backward, 1, 2 and 4 channels
    // a thread at least: 60.1, 60.1, 64.8 us).
    p.k = units <= 16 ? 1 : units <= 32 ? 2 : 4;
    p.waves = (units + p.k - 1) / p.k;
    p.tiles = outer * ((inner + p.lanes * p.vec - 1) / (p.lanes * p.vec));
    if (p.tiles > 0x7fffffffu) return p;
    p.kind = 1;
    const size_t fill = 8192 / p.waves;
    p.partials = (int)(p.tiles < fill ? p.tiles : fill);
    return p;
}

int launched(const char* who) {
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return ggs_fail_(GGS_ERR_HIP, "%s: launch failed: %s", who, hipGetErrorString(e));
    return GGS_OK;
}

template <typename T, int VEC, int LP, int K, bool NT> void planes(bool back, const NormArgs<T>& a, const Plan& p, hipStream_t s) {
    if (back) hipLaunchKernelGGL((k_planes_backward<T, VEC, LP, K, NT>), dim3((unsigned)p.partials), dim3(p.waves * 64), 0, s, a, (unsigned)p.tiles);
    else hipLaunchKernelGGL((k_planes_forward<T, VEC, LP, K, NT>), dim3((unsigned)p.tiles), dim3(p.waves * 64), 0, s, a);
}
template <typename T, int VEC, int LP, bool NT = false> void planes(bool back, const NormArgs<T>& a, const Plan& p, hipStream_t s) {
    if (p.k == 1) planes<T, VEC, LP, 1, NT>(back, a, p, s);
    else if (p.k == 2) planes<T, VEC, LP, 2, NT>(back, a, p, s);
    else planes<T, VEC, LP, 4, NT>(back, a, p, s);
}
// A pass that reads more than this leaves nothing of its inputs in the caches anyway and reads past them: 32 x 1024 x 1024 half
// forward 66.7 -> 60.4 us, 2 x 128 x 256 x 256 float backward 57.7 -> 55.0 us; below, inputs that were just written are still
// there (256 x 128 x 128 float forward 11.7 us, 13.0 us past the caches).
constexpr size_t STREAM_BYTES = (size_t)128 << 20;
template <typename T, int VEC, int G, int K> void rows(bool back, const NormArgs<T>& a, const Plan& p, hipStream_t s) {
    constexpr int THREADS = G > 256 ? G : 256, ROWS = THREADS / G;
    if (back) hipLaunchKernelGGL((k_rows_backward<T, VEC, G, K>), dim3((unsigned)p.partials), dim3(1024), 0, s, a, (unsigned)p.tiles);
    else hipLaunchKernelGGL((k_rows_forward<T, VEC, G, K>), dim3((unsigned)((a.outer + ROWS - 1) / ROWS)), dim3(THREADS), 0, s, a);
}
template <typename T, int VEC, int G> void rows(bool back, const NormArgs<T>& a, const Plan& p, hipStream_t s) {
    if (p.k == 1) rows<T, VEC, G, 1>(back, a, p, s);
    else rows<T, VEC, G, 2>(back, a, p, s);
}

template <typename T> void one_pass(bool back, const NormArgs<T>& a, const Plan& p, hipStream_t s) {
    constexpr int FULL = 16 / sizeof(T);
    if (p.kind == 2) {
        if (p.vec == 1) rows<T, 1, 4>(back, a, p, s);
        else if (p.lanes == 4) rows<T, FULL, 4>(back, a, p, s);
        else if (p.lanes == 16) rows<T, FULL, 16>(back, a, p, s);
        else if (p.lanes == 64) rows<T, FULL, 64>(back, a, p, s);
        else if (p.lanes == 256) rows<T, FULL, 256>(back, a, p, s);
        else if (p.k < 4) rows<T, FULL, 1024>(back, a, p, s);
        else if constexpr (sizeof(T) == 4) rows<T, FULL, 1024, 4>(back, a, p, s);
        return;
    }
    if (p.vec == 1) planes<T, 1, 4>(back, a, p, s);
    else if (p.lanes == 4) planes<T, FULL, 4>(back, a, p, s);
    else if (p.lanes < 64 / FULL) planes<T, FULL, 8>(back, a, p, s);
    else if (a.outer * a.inner * a.C * sizeof(T) * (1 + (a.r != nullptr) + back + (a.gh != nullptr)) < STREAM_BYTES) planes<T, FULL, 64 / FULL>(back, a, p, s);
    else planes<T, FULL, 64 / FULL, true>(back, a, p, s);
}
template <> void one_pass<double>(bool, const NormArgs<double>&, const Plan&, hipStream_t) {}

template <typename T> unsigned two_pass_blocks(const NormArgs<T>& a) {
    const size_t tiles = a.outer * (a.inner == 1 ? 1 : (a.inner + 63) / 64);
    return (unsigned)(tiles < ((size_t)1 << 20) ? tiles : (size_t)1 << 20);
}

// Calls launch(a) for as many maps / rows at a time as a launch may have threads for; `threads` is what one of them takes.
constexpr size_t MAX_THREADS = (size_t)1 << 31;
template <typename T, typename F> int in_parts(const char* who, const NormArgs<T>& all, size_t threads, F&& launch) {
    if (threads > MAX_THREADS) return ggs_fail_(GGS_ERR_SIZE, "%s: more than 2^31 threads for one map", who);
    const size_t per = MAX_THREADS / threads;
    for (size_t o = 0; o < all.outer; o += per) {
        NormArgs<T> a = all;
        a.outer = all.outer - o < per ? all.outer - o : per;
        const size_t at = o * a.C * a.inner;
        a.x += at;
        if (a.r) a.r += at;
        if (a.gy) a.gy += at;
        if (a.gh) a.gh += at;
        if (a.y) a.y += at;
        if (a.h) a.h += at;
        if (a.dx) a.dx += at;
        if (a.q) a.q += o * a.inner;
        launch(a);
        const int rc = launched(who);
        if (rc != GGS_OK) return rc;
    }
    return GGS_OK;
}

template <typename T> int run_forward(NormArgs<T> a, hipStream_t s) {
    const char* who = "ggs_rms_norm_forward";
    const Plan p = plan<T>(a.outer, a.C, a.inner);
    if (p.kind) {
        const size_t threads = p.kind == 2 ? p.lanes : p.tiles / a.outer * p.waves * 64;
        return in_parts(who, a, threads, [&](const NormArgs<T>& b) {
            Plan part = p;
            if (p.kind == 1) part.tiles = p.tiles / a.outer * b.outer;
            one_pass(false, b, part, s);
        });
    }
    if (a.inner == 1) hipLaunchKernelGGL((k_rms_forward<T, false>), dim3(two_pass_blocks(a)), dim3(1024), 0, s, a);
    else hipLaunchKernelGGL((k_rms_forward<T, true>), dim3(two_pass_blocks(a)), dim3(1024), 0, s, a);
    return launched(who);
}

template <typename T, bool SECOND> void launch_dw(const NormArgs<T>& a, hipStream_t s) {
    if (a.inner == 1) hipLaunchKernelGGL((k_rms_dw<T, false, SECOND>), dim3((a.C + 255) / 256, a.n_partial), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_rms_dw<T, true, SECOND>), dim3(a.C, a.n_partial), dim3(256), 0, s, a);
}

// dw from a.n_partial rows of partials (none at all: zeros)
template <typename T> int sum_dw(const char* who, const NormArgs<T>& a, hipStream_t s) {
    hipLaunchKernelGGL((k_rms_dw_sum<T>), dim3((a.C + 7) / 8), dim3(1024), 0, s, a);
    return launched(who);
}

template <typename T> int run_backward(NormArgs<T> a, hipStream_t s) {
    const char* who = "ggs_rms_norm_backward";
    if (a.outer == 0 || a.inner == 0) return a.dw ? sum_dw(who, a, s) : GGS_OK;
    const Plan p = plan<T>(a.outer, a.C, a.inner);
    if (p.kind) {
        one_pass(true, a, p, s);
    } else {
        if (a.inner == 1) hipLaunchKernelGGL((k_rms_backward<T, false>), dim3(two_pass_blocks(a)), dim3(1024), 0, s, a);
        else hipLaunchKernelGGL((k_rms_backward<T, true>), dim3(two_pass_blocks(a)), dim3(1024), 0, s, a);
    }
    int rc = launched(who);
    if (rc != GGS_OK || !a.dw) return rc;
    a.n_partial = p.partials;
    if (!p.kind) launch_dw<T, false>(a, s);
    rc = launched(who);
    return rc != GGS_OK ? rc : sum_dw(who, a, s);
}

template <typename T> int run_second(NormArgs<T> a, hipStream_t s) {
    const char* who = "ggs_rms_norm_double_backward";
    if (a.outer == 0 || a.inner == 0) return a.dw ? sum_dw(who, a, s) : GGS_OK;
    if (a.inner == 1) hipLaunchKernelGGL((k_rms_second<T, false>), dim3(two_pass_blocks(a)), dim3(1024), 0, s, a);
    else hipLaunchKernelGGL((k_rms_second<T, true>), dim3(two_pass_blocks(a)), dim3(1024), 0, s, a);
    int rc = launched(who);
    if (rc != GGS_OK || !a.dw) return rc;
    a.n_partial = two_pass_partials(a.outer, a.inner);
    launch_dw<T, true>(a, s);
    rc = launched(who);
    return rc != GGS_OK ? rc : sum_dw(who, a, s);
}

size_t partials(int dtype, size_t outer, int C, size_t inner) {
    return dtype == GGS_DTYPE_F64 ? plan<double>(outer, C, inner).partials :
           dtype == GGS_DTYPE_F32 ? plan<float>(outer, C, inner).partials : plan<_Float16>(outer, C, inner).partials;
}

int check_sizes(const char* who, int dtype, size_t outer, int channels, size_t inner, double eps) {
    if (dtype < GGS_DTYPE_F32 || dtype > GGS_DTYPE_BF16) return ggs_fail_(GGS_ERR_ARG, "%s: dtype %d is not float / half / double / bfloat16", who, dtype);
    if (channels <= 0) return ggs_fail_(GGS_ERR_ARG, "%s: no channels", who);
    if (channels > 1 << 22) return ggs_fail_(GGS_ERR_SIZE, "%s: more than 2^22 channels", who);
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
    const double least = sizeof(T) == 8 ? 2.3e-308 : 1.2e-38;        // in the normal range: a row of zeros gives zeros, not NaN
    if (a.eps < (typename Acc<T>::type)least) a.eps = (typename Acc<T>::type)least;
    a.inv_c = (typename Acc<T>::type)1 / channels;
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

// Workspace of the double backward pass: b of every pixel, then the partials.
size_t second_bytes(int dtype, size_t outer, int channels, size_t inner) {
    const size_t pixels = outer * inner;
    return (pixels + (size_t)two_pass_partials(outer, inner) * channels) * (dtype == GGS_DTYPE_F64 ? 8 : 4);
}

template <typename T>
int second(size_t outer, int channels, size_t inner, const void* x, const void* residual, const void* weight, int weight_f32, const void* q,
           const void* gy, const void* v, const void* u, void* dh, void* dgy, void* dw, void* workspace, hipStream_t s) {
    NormArgs<T> a = norm_args<T>(outer, channels, inner, x, residual, weight, weight_f32, 0.0);
    a.q = static_cast<typename Acc<T>::type*>(const_cast<void*>(q));
    a.gy = static_cast<const T*>(gy); a.v = static_cast<const T*>(v); a.u = u;
    a.dx = static_cast<T*>(dh); a.dgy = static_cast<T*>(dgy); a.dw = dw;
    a.b = static_cast<typename Acc<T>::type*>(workspace); a.partial = a.b + outer * inner;
    return run_second(a, s);
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
    return partials(dtype, outer, channels, inner) * (size_t)channels * (dtype == GGS_DTYPE_F64 ? 8 : 4);
}

int ggs_rms_norm_backward(int dtype, size_t outer, int channels, size_t inner, const void* x, const void* residual,
                          const void* weight, int weight_f32, const void* q, const void* gy, const void* gh, void* dx,
                          void* dw, void* workspace, size_t workspace_bytes, void* stream) {
    ggs_clear_error_();
    int rc = check_sizes("ggs_rms_norm_backward", dtype, outer, channels, inner, 1.0);
    if (rc != GGS_OK) return rc;
    if (outer && inner && (!x || !q || !gy || !dx)) return ggs_fail_(GGS_ERR_ARG, "ggs_rms_norm_backward: NULL pointer argument");
    const size_t needed = dw ? ggs_rms_norm_workspace_bytes(dtype, outer, channels, inner) : 0;
    if (needed && (!workspace || workspace_bytes < needed))
        return ggs_fail_(GGS_ERR_SIZE, "ggs_rms_norm_backward: the workspace is too small (ggs_rms_norm_workspace_bytes)");
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case GGS_DTYPE_F32: return backward<float>(outer, channels, inner, x, residual, weight, weight_f32, q, gy, gh, dx, dw, workspace, s);
        case GGS_DTYPE_F16: return backward<_Float16>(outer, channels, inner, x, residual, weight, weight_f32, q, gy, gh, dx, dw, workspace, s);
        case GGS_DTYPE_BF16: return backward<__bf16>(outer, channels, inner, x, residual, weight, weight_f32, q, gy, gh, dx, dw, workspace, s);
        default: return backward<double>(outer, channels, inner, x, residual, weight, weight_f32, q, gy, gh, dx, dw, workspace, s);
    }
}

size_t ggs_rms_norm_double_workspace_bytes(int dtype, size_t outer, int channels, size_t inner) {
    return channels <= 0 || outer == 0 || inner == 0 ? 0 : second_bytes(dtype, outer, channels, inner);
}

int ggs_rms_norm_double_backward(int dtype, size_t outer, int channels, size_t inner, const void* x, const void* residual,
                                 const void* weight, int weight_f32, const void* q, const void* gy, const void* v, const void* u,
                                 void* dh, void* dgy, void* dw, void* workspace, size_t workspace_bytes, void* stream) {
    ggs_clear_error_();
    int rc = check_sizes("ggs_rms_norm_double_backward", dtype, outer, channels, inner, 1.0);
    if (rc != GGS_OK) return rc;
    if (outer && inner && (!x || !q || !gy || !dh || !dgy)) return ggs_fail_(GGS_ERR_ARG, "ggs_rms_norm_double_backward: NULL pointer argument");
    if (outer && inner && (!workspace || workspace_bytes < second_bytes(dtype, outer, channels, inner)))
        return ggs_fail_(GGS_ERR_SIZE, "ggs_rms_norm_double_backward: the workspace is too small (ggs_rms_norm_double_workspace_bytes)");
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case GGS_DTYPE_F32: return second<float>(outer, channels, inner, x, residual, weight, weight_f32, q, gy, v, u, dh, dgy, dw, workspace, s);
        case GGS_DTYPE_F16: return second<_Float16>(outer, channels, inner, x, residual, weight, weight_f32, q, gy, v, u, dh, dgy, dw, workspace, s);
        case GGS_DTYPE_BF16: return second<__bf16>(outer, channels, inner, x, residual, weight, weight_f32, q, gy, v, u, dh, dgy, dw, workspace, s);
        default: return second<double>(outer, channels, inner, x, residual, weight, weight_f32, q, gy, v, u, dh, dgy, dw, workspace, s);
    }
}

}  // extern "C"
