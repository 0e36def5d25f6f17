// ggs_gradnorm.hip -- the global gradient norm over many tensors, clipping by it, and the Adam update that reads its gradients
// clipped.  No reference counterpart: the reference's loops clip nothing; their update is ggs_adam.hip's.
//
//   N = sqrt(sum_t sum_i g_ti^2),   c = min(1, max_norm / (N + 1e-6)),   clip: g_ti <- c g_ti,   update: Adam on c g_ti
//
// A first kernel leaves one partial sum of squares per workgroup; every workgroup of the kernel that needs N (the scaling, the
// update) adds those partials up by itself, in one fixed order, so all of them get the same bits and no third launch stands
// between the two.  No atomics: the result does not depend on scheduling.
// Squares are added in DOUBLE: a float square overflows at |g| = 1.8e19 and vanishes below 1e-23, and a float sum over 4e7
// elements is the one place where a training step adds that many numbers.  It costs no time: the gradients arrive at 2
// floats or 3 16-bit values a clock per CU (5.1 and 4.0 TB/s, 256 CUs, 2.4 GHz), and the conversions and fused multiply-adds keep
// the vector pipes busy for 9 % (float) and 19 % (bf16) of the time (VALUBusy, 43.8M gradients).
// HBM-bound: the norm reads every gradient once, the scaling reads and writes it once (nothing when c = 1), the update moves
// ggs_adam.hip's 28 bytes an element.
// Measured (replayed from a graph, inputs of three passes in turn; a copy of 2 GiB runs at 4.9 TB/s here):
//   norm of 43.8M float gradients (78 tensors)           34.6 us: 5.1 TB/s; with the skipped scaling 36.7 us
//   norm and scaling of 43.8M float gradients           102.8 us: 526 MB moved at 5.1 TB/s
//   norm and scaling of 43.8M bf16 gradients             47.3 us: 263 MB moved, the second read from the caches
//   norm and scaling of 6.05M float gradients (7)        16.0 us: two launches and 73 MB
//   norm and update of 43.8M parameters                 281.3 us: 1.40 GB at 5.0 TB/s (torch's clipping and fused Adam: 507 us)
//   norm and update of 36K parameters                     8.0 us: two launches
#include "ggs_kernels.h"

namespace {

#define GGS_NORM_MAX_TENSORS 128          // gradients per launch: a table of 2.7 KB in the kernel arguments
#define GGS_NORM_MAX_BLOCKS 1024          // partial sums per launch
#define GGS_NORM_CHUNK 1024               // 16-byte vectors of one tensor a workgroup takes at a time

struct GradTable {
    unsigned n;
    unsigned end_chunk[GGS_NORM_MAX_TENSORS];     // chunks of tensors 0 .. t; unused entries ~0u
    unsigned char dtype[GGS_NORM_MAX_TENSORS];
    size_t numel[GGS_NORM_MAX_TENSORS];
    void* g[GGS_NORM_MAX_TENSORS];
};

static_assert(sizeof(GradTable) <= 4096 - 64, "the table is a kernel argument");

template <typename T> struct alignas(16) Pack16 { T v[16 / sizeof(T)]; };

// Sum over the 256 threads of the workgroup, the same bits in every thread.
__device__ __forceinline__ double block_sum(double s) {
    __shared__ double part[4];
#pragma unroll
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    return (part[0] + part[1]) + (part[2] + part[3]);
}

// Calls f(packs, store) for a chunk, four packs a thread: all of them on their way before the first is needed where the whole
// chunk lies inside the tensor; in the first and last chunk a pack that reaches over the end is filled element by element (zeros
// outside).  The 16-byte grid is the address space's: a gradient that is a view into a flat bucket starts anywhere.
template <typename T, typename F>
__device__ __forceinline__ void for_chunk(void* ptr, size_t numel, unsigned chunk, F&& f) {
    constexpr int VEC = 16 / sizeof(T);
    const unsigned shift = (unsigned)((reinterpret_cast<uintptr_t>(ptr) & 15) / sizeof(T));
    T* base = static_cast<T*>(ptr) - shift;
    const size_t end = numel + shift, c0 = (size_t)chunk * GGS_NORM_CHUNK;
    Pack16<T> p[4];
    if ((c0 > 0 || shift == 0) && (c0 + GGS_NORM_CHUNK) * VEC <= end) {
        Pack16<T>* at = reinterpret_cast<Pack16<T>*>(base) + c0 + threadIdx.x;
#pragma unroll
        for (int k = 0; k < 4; ++k) p[k] = at[k * 256];
        f(p, [&](int k, const Pack16<T>& q) { at[k * 256] = q; });
    } else {
        const auto whole = [&](size_t e) { return (e > 0 || shift == 0) && e + VEC <= end; };
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const size_t e = (c0 + threadIdx.x + k * 256) * VEC;
            if (whole(e)) p[k] = *reinterpret_cast<Pack16<T>*>(base + e);
            else for (int j = 0; j < VEC; ++j) p[k].v[j] = e + j >= shift && e + j < end ? base[e + j] : (T)0.0f;
        }
        f(p, [&](int k, const Pack16<T>& q) {
            const size_t e = (c0 + threadIdx.x + k * 256) * VEC;
            if (whole(e)) *reinterpret_cast<Pack16<T>*>(base + e) = q;
            else for (int j = 0; j < VEC; ++j) if (e + j >= shift && e + j < end) base[e + j] = q.v[j];
        });
    }
}

// The tensor of chunk c: the number of tensors that end at or before it (two entries of end_chunk a lane).
struct Finder {
    unsigned e0, e1;
    __device__ __forceinline__ explicit Finder(const GradTable& t) : e0(t.end_chunk[threadIdx.x & 63]), e1(t.end_chunk[64 + (threadIdx.x & 63)]) {}
    __device__ __forceinline__ int operator()(unsigned c) const {
        return __builtin_amdgcn_readfirstlane((int)(__popcll(__ballot(e0 <= c)) + __popcll(__ballot(e1 <= c))));
    }
};

template <typename T>
__device__ __forceinline__ double chunk_squares(void* g, size_t numel, unsigned chunk) {
    double s[4] = {};
    for_chunk<T>(g, numel, chunk, [&](const Pack16<T> (&p)[4], auto&&) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
#pragma unroll
            for (int j = 0; j < (int)(16 / sizeof(T)); ++j) { const double d = (double)(float)p[k].v[j]; s[k] = fma(d, d, s[k]); }
        }
    });
    return (s[0] + s[1]) + (s[2] + s[3]);
}

// 1024 workgroups: 256 / 512 / 2048 take 63.7 / 40.9 / 39.4 us for 43.8M float gradients, 1024 take 36.4.
__global__ __launch_bounds__(256) void k_grad_squares(GradTable t, double* partial) {
    const Finder find(t);
    const unsigned total = t.end_chunk[t.n - 1];
    double s = 0.0;
    for (unsigned c = blockIdx.x; c < total; c += gridDim.x) {
        const int i = find(c);
        const unsigned chunk = c - (i ? t.end_chunk[i - 1] : 0);
        switch (t.dtype[i]) {
            case GGS_DTYPE_F32: s += chunk_squares<float>(t.g[i], t.numel[i], chunk); break;
            case GGS_DTYPE_F16: s += chunk_squares<_Float16>(t.g[i], t.numel[i], chunk); break;
            default: s += chunk_squares<__bf16>(t.g[i], t.numel[i], chunk); break;
        }
    }
    s = block_sum(s);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// N from the partial sums (256 threads, fixed order)
__device__ __forceinline__ double norm_of(const double* partial, int n) {
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 256) s += partial[i];
    return sqrt(block_sum(s));
}

// torch.nn.utils.clip_grad_norm_'s factor: a NaN norm gives NaN, an infinite one 0
__device__ __forceinline__ float clip_factor(double norm, double max_norm) {
    const double c = max_norm / (norm + 1e-6);
    return c > 1.0 ? 1.0f : (float)c;
}

// guard (NULL: none): a word that voids the write
__global__ __launch_bounds__(256) void k_grad_norm(const double* partial, int n, float* norm, const unsigned long long* guard) {
    if (guard && *guard) return;
    const double d = norm_of(partial, n);
    if (threadIdx.x == 0) *norm = (float)d;
}

template <typename T>
__device__ __forceinline__ void chunk_scale(void* g, size_t numel, unsigned chunk, float c) {
    for_chunk<T>(g, numel, chunk, [&](Pack16<T> (&p)[4], auto&& store) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
#pragma unroll
            for (int j = 0; j < (int)(16 / sizeof(T)); ++j) p[k].v[j] = (T)((float)p[k].v[j] * c);
            store(k, p[k]);
        }
    });
}

__global__ __launch_bounds__(256) void k_grad_scale(GradTable t, const double* partial, int n_partial, double max_norm, float* norm) {
    const double d = norm_of(partial, n_partial);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)d;
    const float f = clip_factor(d, max_norm);
    if (f == 1.0f) return;                                        // x * 1 = x: nothing to write (a NaN is not equal to 1)
    const Finder find(t);
    const unsigned total = t.end_chunk[t.n - 1];
    for (unsigned c = blockIdx.x; c < total; c += gridDim.x) {
        const int i = find(c);
        const unsigned chunk = c - (i ? t.end_chunk[i - 1] : 0);
        switch (t.dtype[i]) {
            case GGS_DTYPE_F32: chunk_scale<float>(t.g[i], t.numel[i], chunk, f); break;
            case GGS_DTYPE_F16: chunk_scale<_Float16>(t.g[i], t.numel[i], chunk, f); break;
            default: chunk_scale<__bf16>(t.g[i], t.numel[i], chunk, f); break;
        }
    }
}

// ---- the clipped update ---------------------------------------------------------------------------------------------------
#define GGS_CLIP_MAX_TENSORS 64           // a table of 3.9 KB
#define GGS_CLIP_BLOCKS 2048              // workgroups a launch, about
struct ClipAdam {
    int n, tick;
    unsigned first_block[GGS_CLIP_MAX_TENSORS + 1];
    size_t numel[GGS_CLIP_MAX_TENSORS];
    float* p[GGS_CLIP_MAX_TENSORS]; const float* g[GGS_CLIP_MAX_TENSORS];
    float* m[GGS_CLIP_MAX_TENSORS]; float* v[GGS_CLIP_MAX_TENSORS];
    const float* lr[GGS_CLIP_MAX_TENSORS];
    AdamState* s[GGS_CLIP_MAX_TENSORS];
    const unsigned long long* guard;
    const double* partial; int n_partial; double max_norm; float* norm;
    float beta2, omb1, omb2, eps;
    double beta1d, beta2d;
};

static_assert(sizeof(ClipAdam) <= 4096, "the table is a kernel argument");

// ggs_adam.hip's update (torch's single-tensor Adam) with the gradient scaled first
__device__ __forceinline__ void adam1(float& p, float g, float& m, float& v, const ClipAdam& a, float step_size, float bias2_sqrt) {
    m = fmaf(a.omb1, g - m, m);
    v = fmaf(a.omb2, g * g, v * a.beta2);
    p = fmaf(-step_size, m / (sqrtf(v) / bias2_sqrt + a.eps), p);
}

// Parameters and moments pass by the caches in both directions: they come back a step later, and what they would push out is the
// gradient the norm has just read (43.8M parameters, norm and update: 309 -> 280 us; 6M: 50.0 -> 48.7 us).
typedef float Float4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ float4 load_past(const float4* p) {
    const Float4 v = __builtin_nontemporal_load(reinterpret_cast<const Float4*>(p));
    return make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store_past(float4* p, const float4& a) {
    const Float4 v = {a.x, a.y, a.z, a.w};
    __builtin_nontemporal_store(v, reinterpret_cast<Float4*>(p));
}
struct AdamVec { float4 p, g, m, v; };

__global__ __launch_bounds__(256) void k_adam_clip(ClipAdam a) {
    if (a.guard && *a.guard) return;
    const int l = threadIdx.x & 63;
    const unsigned end_block = l < a.n ? a.first_block[l + 1] : ~0u;
    const int t = __builtin_amdgcn_readfirstlane((int)__popcll(__ballot(end_block <= blockIdx.x)));
    const unsigned b0 = a.first_block[t], nb = a.first_block[t + 1] - b0;
    const size_t n = a.numel[t], n4 = n / 4, stride = (size_t)nb * 256;
    float4* p4 = reinterpret_cast<float4*>(a.p[t]);
    const float4* g4 = reinterpret_cast<const float4*>(a.g[t]);
    float4* m4 = reinterpret_cast<float4*>(a.m[t]);
    float4* v4 = reinterpret_cast<float4*>(a.v[t]);
    size_t i = (size_t)(blockIdx.x - b0) * 256 + threadIdx.x;
    AdamVec now, next;                       // one iteration ahead: the first loads run beside the sum of the partials
    if (i < n4) now = {load_past(p4 + i), g4[i], load_past(m4 + i), load_past(v4 + i)};
    AdamState* st = a.s[t];
    float bias1 = st->bias1, bs = st->bias2_sqrt;
    long long tt = 0;
    double p1 = 0.0, p2 = 0.0;
    if (a.tick) {                                                        // ggs_adam_tick_one, without the stores
        tt = st->step + 1;
        p1 = tt == 1 ? a.beta1d : st->pow1 * a.beta1d;
        p2 = tt == 1 ? a.beta2d : st->pow2 * a.beta2d;
        bias1 = (float)(1.0 - p1);
        bs = (float)sqrt(1.0 - p2);
    }
    const float step_size = *a.lr[t] / bias1;
    const double d = norm_of(a.partial, a.n_partial);
    if (a.norm && blockIdx.x == 0 && threadIdx.x == 0) *a.norm = (float)d;
    const float f = clip_factor(d, a.max_norm);
    for (; i < n4; i += stride, now = next) {
        const size_t j = i + stride;
        if (j < n4) next = {load_past(p4 + j), g4[j], load_past(m4 + j), load_past(v4 + j)};
        adam1(now.p.x, now.g.x * f, now.m.x, now.v.x, a, step_size, bs);
        adam1(now.p.y, now.g.y * f, now.m.y, now.v.y, a, step_size, bs);
        adam1(now.p.z, now.g.z * f, now.m.z, now.v.z, a, step_size, bs);
        adam1(now.p.w, now.g.w * f, now.m.w, now.v.w, a, step_size, bs);
        store_past(p4 + i, now.p); store_past(m4 + i, now.m); store_past(v4 + i, now.v);
    }
    if (blockIdx.x == b0 && threadIdx.x < (n & 3)) {
        const size_t k = n4 * 4 + threadIdx.x;
        adam1(a.p[t][k], a.g[t][k] * f, a.m[t][k], a.v[t][k], a, step_size, bs);
    }
    if (a.tick) __syncthreads();             // every wave of this workgroup has read the state (its values fed the loop above)
    if (a.tick && threadIdx.x == 0) {        // as in ggs_adam.hip: the last workgroup of a tensor stores the advanced state
        if (atomicAdd(&st->ticket, 1u) == nb - 1) {
            st->step = tt; st->pow1 = p1; st->pow2 = p2; st->bias1 = bias1; st->bias2_sqrt = bs;
            atomicExch(&st->ticket, 0u);
        }
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------------
inline size_t elem_size(int dtype) { return dtype == GGS_DTYPE_F32 ? 4 : dtype == GGS_DTYPE_F16 || dtype == GGS_DTYPE_BF16 ? 2 : 0; }

int check_grads(const char* who, int n, const size_t* numel, const void* const* grads, const int* dtypes) {
    if (n < 0) return ggs_fail_(GGS_ERR_ARG, "%s: negative number of tensors", who);
    if (n > 0 && (!numel || !grads)) return ggs_fail_(GGS_ERR_ARG, "%s: NULL pointer argument", who);
    for (int i = 0; i < n; ++i) {
        if (numel[i] == 0) continue;
        const size_t es = elem_size(dtypes ? dtypes[i] : GGS_DTYPE_F32);
        if (!es) return ggs_fail_(GGS_ERR_ARG, "%s: dtype %d is not float / half / bfloat16", who, dtypes[i]);
        if (!grads[i]) return ggs_fail_(GGS_ERR_ARG, "%s: NULL tensor pointer", who);
        if (reinterpret_cast<uintptr_t>(grads[i]) % es) return ggs_fail_(GGS_ERR_ARG, "%s: a tensor is not aligned to its element size", who);
        if (numel[i] > ((size_t)1 << 40)) return ggs_fail_(GGS_ERR_SIZE, "%s: more than 2^40 elements in a tensor", who);
    }
    return GGS_OK;
}

// Fills `t` with the non-empty tensors from `i` on (as many as fit) and advances `i`; false: none left.
bool next_table(GradTable& t, int& i, int n, const size_t* numel, const void* const* grads, const int* dtypes) {
    t.n = 0;
    size_t total = 0;
    for (; i < n && t.n < GGS_NORM_MAX_TENSORS; ++i) {
        if (numel[i] == 0) continue;
        const int dt = dtypes ? dtypes[i] : GGS_DTYPE_F32;
        const size_t es = elem_size(dt), vec = 16 / es, shift = (reinterpret_cast<uintptr_t>(grads[i]) & 15) / es;
        const size_t chunks = ((numel[i] + shift + vec - 1) / vec + GGS_NORM_CHUNK - 1) / GGS_NORM_CHUNK;
        if (total + chunks > 0x7fffffffu) break;                  // (one tensor alone has at most 2^28 chunks)
        total += chunks;
        t.end_chunk[t.n] = (unsigned)total;
        t.dtype[t.n] = (unsigned char)dt;
        t.numel[t.n] = numel[i];
        t.g[t.n] = const_cast<void*>(grads[i]);
        ++t.n;
    }
    for (unsigned k = t.n; k < GGS_NORM_MAX_TENSORS; ++k) t.end_chunk[k] = ~0u;
    return t.n > 0;
}

// The partial sums of all tensors; *n_partial of them.
int launch_squares(const char* who, int n, const size_t* numel, const void* const* grads, const int* dtypes, void* workspace,
                   size_t workspace_bytes, int* n_partial, hipStream_t s) {
    *n_partial = 0;
    GradTable t;
    for (int i = 0; next_table(t, i, n, numel, grads, dtypes);) {
        const unsigned total = t.end_chunk[t.n - 1], blocks = total < GGS_NORM_MAX_BLOCKS ? total : GGS_NORM_MAX_BLOCKS;
        if (!workspace || ((size_t)*n_partial + blocks) * sizeof(double) > workspace_bytes)
            return ggs_fail_(GGS_ERR_SIZE, "%s: the workspace is too small (ggs_grad_norm_workspace_bytes)", who);
        hipLaunchKernelGGL(k_grad_squares, dim3(blocks), dim3(256), 0, s, t, static_cast<double*>(workspace) + *n_partial);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess) return ggs_fail_(GGS_ERR_HIP, "%s: launch failed: %s", who, hipGetErrorString(e));
        *n_partial += (int)blocks;
    }
    return GGS_OK;
}

int launch_norm(const char* who, const void* workspace, int n_partial, float* norm, const void* guard, hipStream_t s) {
    hipLaunchKernelGGL(k_grad_norm, dim3(1), dim3(256), 0, s, static_cast<const double*>(workspace), n_partial, norm,
                       static_cast<const unsigned long long*>(guard));
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return ggs_fail_(GGS_ERR_HIP, "%s: launch failed: %s", who, hipGetErrorString(e));
    return GGS_OK;
}

}  // namespace

extern "C" {

size_t ggs_grad_norm_workspace_bytes(int n_tensors) {
    return n_tensors <= 0 ? 0 : ((size_t)(n_tensors - 1) / GGS_NORM_MAX_TENSORS + 1) * GGS_NORM_MAX_BLOCKS * sizeof(double);
}

int ggs_grad_norm(int n_tensors, const size_t* numel, const void* const* grads, const int* dtypes, float* norm,
                  void* workspace, size_t workspace_bytes, void* stream) {
    ggs_clear_error_();
    int rc = check_grads("ggs_grad_norm", n_tensors, numel, grads, dtypes), n_partial = 0;
    if (rc != GGS_OK) return rc;
    if (!norm) return ggs_fail_(GGS_ERR_ARG, "ggs_grad_norm: NULL norm");
    rc = launch_squares("ggs_grad_norm", n_tensors, numel, grads, dtypes, workspace, workspace_bytes, &n_partial, (hipStream_t)stream);
    return rc != GGS_OK ? rc : launch_norm("ggs_grad_norm", workspace, n_partial, norm, nullptr, (hipStream_t)stream);
}

int ggs_grad_clip(int n_tensors, const size_t* numel, void* const* grads, const int* dtypes, double max_norm, float* norm,
                  void* workspace, size_t workspace_bytes, void* stream) {
    ggs_clear_error_();
    int rc = check_grads("ggs_grad_clip", n_tensors, numel, grads, dtypes), n_partial = 0;
    if (rc != GGS_OK) return rc;
    if (!norm) return ggs_fail_(GGS_ERR_ARG, "ggs_grad_clip: NULL norm");
    if (!(max_norm >= 0.0)) return ggs_fail_(GGS_ERR_ARG, "ggs_grad_clip: max_norm must not be negative");
    hipStream_t s = (hipStream_t)stream;
    rc = launch_squares("ggs_grad_clip", n_tensors, numel, grads, dtypes, workspace, workspace_bytes, &n_partial, s);
    if (rc != GGS_OK) return rc;
    if (n_partial == 0) return launch_norm("ggs_grad_clip", workspace, 0, norm, nullptr, s);
    GradTable t;
    bool first = true;
    for (int i = 0; next_table(t, i, n_tensors, numel, grads, dtypes); first = false) {
        const unsigned total = t.end_chunk[t.n - 1], blocks = total < 2048 ? total : 2048;
        hipLaunchKernelGGL(k_grad_scale, dim3(blocks), dim3(256), 0, s, t, static_cast<const double*>(workspace), n_partial,
                           max_norm, first ? norm : nullptr);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess) return ggs_fail_(GGS_ERR_HIP, "ggs_grad_clip: launch failed: %s", hipGetErrorString(e));
    }
    return GGS_OK;
}

int ggs_adam_clip_step(int n_tensors, const size_t* numel, float* const* params, const float* const* grads,
                       float* const* exp_avgs, float* const* exp_avg_sqs, const float* const* lrs, void* const* states,
                       double beta1, double beta2, double eps, double max_norm, int tick, const void* guard, float* norm,
                       void* workspace, size_t workspace_bytes, void* stream) {
    ggs_clear_error_();
    const void* const* gv = reinterpret_cast<const void* const*>(grads);
    int rc = check_grads("ggs_adam_clip_step", n_tensors, numel, gv, nullptr), n_partial = 0;
    if (rc != GGS_OK) return rc;
    if (!norm) return ggs_fail_(GGS_ERR_ARG, "ggs_adam_clip_step: NULL norm");
    if (!(max_norm >= 0.0)) return ggs_fail_(GGS_ERR_ARG, "ggs_adam_clip_step: max_norm must not be negative");
    if (n_tensors > 0 && (!params || !exp_avgs || !exp_avg_sqs || !lrs || !states))
        return ggs_fail_(GGS_ERR_ARG, "ggs_adam_clip_step: NULL pointer argument");
    for (int i = 0; i < n_tensors; ++i) {
        if (numel[i] == 0) continue;
        if (!params[i] || !exp_avgs[i] || !exp_avg_sqs[i] || !lrs[i] || !states[i])
            return ggs_fail_(GGS_ERR_ARG, "ggs_adam_clip_step: NULL tensor pointer");
        if ((reinterpret_cast<uintptr_t>(params[i]) | reinterpret_cast<uintptr_t>(grads[i]) |
             reinterpret_cast<uintptr_t>(exp_avgs[i]) | reinterpret_cast<uintptr_t>(exp_avg_sqs[i])) & 15)
            return ggs_fail_(GGS_ERR_ARG, "ggs_adam_clip_step: tensors must be 16-byte aligned");
    }
    hipStream_t s = (hipStream_t)stream;
    rc = launch_squares("ggs_adam_clip_step", n_tensors, numel, gv, nullptr, workspace, workspace_bytes, &n_partial, s);
    if (rc != GGS_OK) return rc;
    if (n_partial == 0) return launch_norm("ggs_adam_clip_step", workspace, 0, norm, guard, s);
    ClipAdam a;
    a.tick = tick; a.guard = static_cast<const unsigned long long*>(guard);
    a.partial = static_cast<const double*>(workspace); a.n_partial = n_partial; a.max_norm = max_norm; a.norm = norm;
    a.beta2 = (float)beta2; a.omb1 = (float)(1.0 - beta1); a.omb2 = (float)(1.0 - beta2); a.eps = (float)eps;
    a.beta1d = beta1; a.beta2d = beta2;
    for (int i = 0; i < n_tensors;) {
        int end = i;                                              // the tensors of this launch
        size_t total = 0;
        for (int k = 0; end < n_tensors && k < GGS_CLIP_MAX_TENSORS; ++end) {
            k += numel[end] != 0;
            total += numel[end];
        }
        // vectors a workgroup takes: enough of them that adding up the partials is a small part of its work
        const size_t share = total / 4 / GGS_CLIP_BLOCKS < 256 ? 256 : total / 4 / GGS_CLIP_BLOCKS;
        a.n = 0; a.first_block[0] = 0;
        for (; i < end; ++i) {
            if (numel[i] == 0) continue;
            const int k = a.n++;
            a.numel[k] = numel[i]; a.p[k] = params[i]; a.g[k] = grads[i]; a.m[k] = exp_avgs[i]; a.v[k] = exp_avg_sqs[i];
            a.lr[k] = lrs[i]; a.s[k] = static_cast<AdamState*>(states[i]);
            a.first_block[k + 1] = a.first_block[k] + (unsigned)(numel[i] / 4 < share ? 1 : (numel[i] / 4 + share - 1) / share);
        }
        if (a.n == 0) break;
        hipLaunchKernelGGL(k_adam_clip, dim3(a.first_block[a.n]), dim3(256), 0, s, a);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess) return ggs_fail_(GGS_ERR_HIP, "ggs_adam_clip_step: launch failed: %s", hipGetErrorString(e));
        a.norm = nullptr;
    }
    return GGS_OK;
}

}  // extern "C"
