// Norm of many gradients taken as one vector, and their scaling by min(1, max_norm / (norm + 1e-6)).
//
// Two launches for (up to) 280 tensors, whatever their sizes (176 where the results go to other tensors): the first sums |g|^p into
// one double per workgroup, the second adds those sums in their order -- every workgroup for itself, 8 KB that sit in L2 -- and
// scales.  Both are bound by the bytes of the gradients: the factor needs the norm of all of them, so they are read twice (unless
// they are in place and the factor is 1).  Sums are doubles from the first element on: a square of an fp32 gradient may leave fp32's
// range, and a sum over 10^8 elements needs more than 24 bits.  No atomics: the result does not depend on the order in which
// workgroups run.
//
// 2^29 elements in 64 tensors: the norm 6.1 TB/s (fp32 351 us, bf16 175), the norm and the scaled copy 5.4 and 5.2 TB/s over the
// three passes (1185 and 617 us).  Below about 30 MB the launches and the host's walk over the list are longer than the bytes:
// 31 chunks of a head's gradients 10 us, 111 tensors of 7 M fp16 values 24 us (the two kernels 19), 201 of 76 M bf16 values below the
// limit 34 (33).
// Every scaling launch adds the sums of the whole list, so that part grows with the square of the number of launches: 4096 fp32
// values each, into other tensors (us, in a graph): 600 tensors 34, 2000 121, 5000 303, 20000 1766.
#include "../../include/dethead.h"
#include "dh_common.h"
#include <algorithm>

namespace {

constexpr int READ = 280, BOTH = 176;       // tensors of one launch: the table travels as a kernel argument (4 KB at most)
constexpr int CHUNK = 8192;         // elements a workgroup takes at a time
constexpr int GROUPS = 1024;        // workgroups of a launch at most: 4 per CU

// OUT: with other tensors for the results; without, what is read is what is written.
template <bool OUT> struct Table {
    static constexpr int SIZE = OUT ? BOTH : READ;
    void* in[SIZE];
    void* to[OUT ? SIZE : 1];
    int first[SIZE + 1];            // first chunk of each tensor
    uint16_t tail[SIZE];            // elements of each tensor's last chunk
    int count;

    __device__ void* out(int k) const { return OUT ? to[k] : in[k]; }
    __device__ int length(int k, int chunk) const { return chunk + 1 < first[k + 1] ? CHUNK : tail[k]; }
};
static_assert(sizeof(Table<true>) <= 4096 - 64 && sizeof(Table<false>) <= 4096 - 64, "beside the other arguments");
static_assert(CHUNK < 65536, "a tail has 16 bits");

template <typename T> __device__ __forceinline__ float up(T v) { return (float)v; }

// |g|^p into the running value; the maximum keeps a NaN once it has met one
template <int KIND> __device__ __forceinline__ double join(double a, double b)
{
    if (KIND == DH_NORM_MAX) return (b > a || b != b) ? b : a;
    return a + b;
}
template <int KIND> __device__ __forceinline__ double power(float g)
{
    const double d = (double)g;
    return KIND == DH_NORM_2 ? d * d : (d < 0 ? -d : d);
}

template <int KIND> __device__ __forceinline__ double wave_join(double v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = join<KIND>(v, __shfl_xor(v, o, 64));
    return v;
}

// the same value in every thread of the workgroup, joined in a fixed order
template <int KIND> __device__ __forceinline__ double group_join(double v, double* shared)
{
    v = wave_join<KIND>(v);
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    return join<KIND>(join<KIND>(shared[0], shared[1]), join<KIND>(shared[2], shared[3]));
}

template <bool OUT> __device__ __forceinline__ int find(const Table<OUT>& t, int chunk)
{
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= chunk) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// A workgroup's chunks, `begin` to `end`: consecutive ones, so that the table is searched once and then followed.
struct Run {
    int begin, end, k;
};
template <bool OUT> __device__ __forceinline__ Run run_of(const Table<OUT>& t)
{
    const int64_t all = t.first[t.count];
    const int begin = (int)(all * blockIdx.x / gridDim.x), end = (int)(all * (blockIdx.x + 1) / gridDim.x);
    return {begin, end, find(t, begin)};
}

template <typename T, int KIND>
__global__ void __launch_bounds__(256) k_grad_power(const Table<false> t, double* __restrict__ partial)
{
    constexpr int V = 16 / sizeof(T);
    __shared__ double shared[4];
    double sum = 0.0;
    Run run = run_of(t);
    for (int c = run.begin; c < run.end; ++c) {
        while (c >= t.first[run.k + 1]) ++run.k;
        const int k = run.k;
        const int64_t at = (int64_t)(c - t.first[k]) * CHUNK;
        const T* g = (const T*)t.in[k] + at;
        const int n = t.length(k, c);
        if (n == CHUNK) {               // all of a full chunk's pieces are requested at once
            constexpr int N = CHUNK / (256 * V);
            T v[N][V];
#pragma unroll
            for (int u = 0; u < N; ++u) __builtin_memcpy(v[u], g + (u * 256 + threadIdx.x) * V, 16);
#pragma unroll
            for (int u = 0; u < N; ++u)
#pragma unroll
                for (int e = 0; e < V; ++e) sum = join<KIND>(sum, power<KIND>(up(v[u][e])));
            continue;
        }
        for (int i = threadIdx.x * V; i < n; i += 256 * V) {
            T v[V];
            if (i + V <= n) __builtin_memcpy(v, g + i, 16);
            else
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] = i + e < n ? g[i + e] : T(0);
#pragma unroll
            for (int e = 0; e < V; ++e) sum = join<KIND>(sum, power<KIND>(up(v[e])));
        }
    }
    sum = group_join<KIND>(sum, shared);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// the norm from the partial sums
template <int KIND> __device__ __forceinline__ double total(const double* __restrict__ partial, int parts, double* shared)
{
    double sum = 0.0;
    for (int i = threadIdx.x; i < parts; i += 256 * 8) {        // eight requested at once: a trip to L2 each is what this costs
        double v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = i + 256 * u < parts ? partial[i + 256 * u] : 0.0;
#pragma unroll
        for (int u = 0; u < 8; ++u) sum = join<KIND>(sum, v[u]);
    }
    return group_join<KIND>(sum, shared);
}

template <int KIND>
__global__ void __launch_bounds__(256) k_grad_join(const double* __restrict__ partial, int parts, const float* __restrict__ scale,
                                                   double* __restrict__ sum, float* __restrict__ norm)
{
    __shared__ double shared[4];
    const double v = total<KIND>(partial, parts, shared);
    if (threadIdx.x == 0) {
        if (sum) *sum = v;
        if (norm) *norm = (float)((KIND == DH_NORM_2 ? sqrt(v) : v) / (scale ? fabs((double)*scale) : 1.0));
    }
}

template <typename T, typename U, int KIND, bool OUT>
__global__ void __launch_bounds__(256) k_grad_clip(const Table<OUT> t, const double* __restrict__ partial, int parts,
                                                   const float* __restrict__ scale, double max_norm, float* __restrict__ norm)
{
    constexpr int V = 16 / sizeof(T);
    __shared__ double shared[4];
    const double sum = total<KIND>(partial, parts, shared);
    const double by = scale ? (double)*scale : 1.0;
    const double n_all = (KIND == DH_NORM_2 ? sqrt(sum) : sum) / fabs(by);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n_all;
    double factor = max_norm / (n_all + 1e-6);
    factor = factor > 1.0 ? 1.0 : factor;               // (a NaN norm leaves a NaN factor)
    // as two floats: a factor near the end of fp32's range (norms of 1e38 do not leave it) would lose its bits in one
    const double both = factor / by;
    const float f2 = fabs(both) < 0x1p-100 ? 0x1p-64f : 1.f, f = (float)(f2 == 1.f ? both : both * 0x1p64);
    if (!OUT && f == 1.f && f2 == 1.f) return;
    Run run = run_of(t);
    for (int c = run.begin; c < run.end; ++c) {
        while (c >= t.first[run.k + 1]) ++run.k;
        const int k = run.k;
        if (f == 1.f && f2 == 1.f && t.in[k] == t.out(k)) continue;   // in place and nothing to do
        const int64_t at = (int64_t)(c - t.first[k]) * CHUNK;
        const T* g = (const T*)t.in[k] + at;
        U* o = (U*)t.out(k) + at;
        const int n = t.length(k, c);
        if (n == CHUNK) {
            constexpr int N = CHUNK / (256 * V);
            T v[N][V];
#pragma unroll
            for (int u = 0; u < N; ++u) __builtin_memcpy(v[u], g + (u * 256 + threadIdx.x) * V, 16);
#pragma unroll
            for (int u = 0; u < N; ++u) {
                U w[V];
#pragma unroll
                for (int e = 0; e < V; ++e) w[e] = (U)(up(v[u][e]) * f * f2);
                __builtin_memcpy(o + (u * 256 + threadIdx.x) * V, w, sizeof(w));
            }
            continue;
        }
        for (int i = threadIdx.x * V; i < n; i += 256 * V) {
            T v[V];
            U w[V];
            if (i + V <= n) {
                __builtin_memcpy(v, g + i, 16);
#pragma unroll
                for (int e = 0; e < V; ++e) w[e] = (U)(up(v[e]) * f * f2);
                __builtin_memcpy(o + i, w, sizeof(w));
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (i + e < n) o[i + e] = (U)(up(g[i + e]) * f * f2);
            }
        }
    }
}

int groups_of(int chunks) { return chunks < GROUPS ? chunks : GROUPS; }

int64_t chunks_of(const int64_t* n, int lo, int hi)
{
    int64_t c = 0;
    for (int k = lo; k < hi; ++k) c += (n[k] + CHUNK - 1) / CHUNK;
    return c;
}

// the table of tensors lo.. and how many chunks it has (sized() has bounded them)
template <bool OUT>
int fill(Table<OUT>* t, const void* const* in, void* const* out, const int64_t* n, int lo, int count)
{
    const int hi = lo + t->SIZE < count ? lo + t->SIZE : count;
    int64_t c = 0;
    for (int k = lo; k < hi; ++k) {
        t->in[k - lo] = (void*)in[k];
        if (OUT) t->to[k - lo] = out[k];
        t->first[k - lo] = (int)c;
        t->tail[k - lo] = (uint16_t)(n[k] ? (n[k] - 1) % CHUNK + 1 : 0);
        c += (n[k] + CHUNK - 1) / CHUNK;
    }
    t->count = hi - lo;
    t->first[hi - lo] = (int)c;
    return (int)c;
}

bool sized(const int64_t* n, int count)
{
    if (count < 0 || (count > 0 && !n)) return false;
    int64_t chunks = 0;                     // chunk numbers and their strides stay within an int
    for (int k = 0; k < count; ++k) {
        if (n[k] < 0 || n[k] >= (1ll << 40)) return false;
        chunks += (n[k] + CHUNK - 1) / CHUNK;
        if (chunks >= (1ll << 30)) return false;
    }
    return true;
}

template <typename T, int KIND>
void launch_power(const Table<false>& t, int groups, double* partial, hipStream_t st)
{
    hipLaunchKernelGGL((k_grad_power<T, KIND>), dim3((unsigned)groups), dim3(256), 0, st, t, partial);
}

template <typename T>
void launch_power(const Table<false>& t, int kind, int groups, double* partial, hipStream_t st)
{
    if (kind == DH_NORM_1) launch_power<T, DH_NORM_1>(t, groups, partial, st);
    else if (kind == DH_NORM_2) launch_power<T, DH_NORM_2>(t, groups, partial, st);
    else launch_power<T, DH_NORM_MAX>(t, groups, partial, st);
}

template <typename T, typename U, bool OUT>
void launch_clip(const Table<OUT>& t, int kind, int groups, const double* partial, int parts, const float* scale, double max_norm, float* norm,
                 hipStream_t st)
{
    const dim3 grid((unsigned)groups), block(256);
    if (kind == DH_NORM_1) hipLaunchKernelGGL((k_grad_clip<T, U, DH_NORM_1, OUT>), grid, block, 0, st, t, partial, parts, scale, max_norm, norm);
    else if (kind == DH_NORM_2) hipLaunchKernelGGL((k_grad_clip<T, U, DH_NORM_2, OUT>), grid, block, 0, st, t, partial, parts, scale, max_norm, norm);
    else hipLaunchKernelGGL((k_grad_clip<T, U, DH_NORM_MAX, OUT>), grid, block, 0, st, t, partial, parts, scale, max_norm, norm);
}

// All tensors of a list; whether there were any elements.  `norm` receives its value from the first launch.
template <bool OUT>
bool clip_all(const void* const* grads, void* const* out, const int64_t* n, int count, int dtype, int out_dtype, int kind, const double* partial,
              int parts, const float* scale, double max_norm, float* norm, hipStream_t st)
{
    bool told = false;
    for (int lo = 0; lo < count; lo += Table<OUT>::SIZE) {
        Table<OUT> t;
        const int chunks = fill(&t, grads, out, n, lo, count);
        if (chunks == 0) continue;
        const int groups = groups_of(chunks);
        float* say = told ? nullptr : norm;
        told = true;
        if (dtype == DH_F32) launch_clip<float, float>(t, kind, groups, partial, parts, scale, max_norm, say, st);
        else if (dtype == DH_F16 && out_dtype == DH_F16) launch_clip<_Float16, _Float16>(t, kind, groups, partial, parts, scale, max_norm, say, st);
        else if (dtype == DH_BF16 && out_dtype == DH_BF16) launch_clip<__bf16, __bf16>(t, kind, groups, partial, parts, scale, max_norm, say, st);
        else if constexpr (OUT) {
            if (dtype == DH_F16) launch_clip<_Float16, float>(t, kind, groups, partial, parts, scale, max_norm, say, st);
            else launch_clip<__bf16, float>(t, kind, groups, partial, parts, scale, max_norm, say, st);
        }
    }
    return told;
}

bool types(int dtype) { return dtype >= DH_F32 && dtype <= DH_BF16; }
bool kinds(int kind) { return kind == DH_NORM_1 || kind == DH_NORM_2 || kind == DH_NORM_MAX; }

}  // namespace

extern "C" int64_t dh_grad_parts(const int64_t* n, int count)
{
    if (!sized(n, count)) return 0;
    int64_t parts = 0;
    for (int lo = 0; lo < count; lo += READ) {
        const int hi = lo + READ < count ? lo + READ : count;
        const int64_t c = chunks_of(n, lo, hi);
        parts += c < GROUPS ? c : GROUPS;
    }
    return parts;
}

extern "C" int dh_grad_power(const void* const* grads, const int64_t* n, int count, int dtype, int norm, double* partial, int64_t parts,
                             void* stream)
{
    if (!sized(n, count) || (count && !grads) || !types(dtype) || !kinds(norm)) return DH_ERR_ARG;
    for (int k = 0; k < count; ++k) {
        if (n[k] && !grads[k]) return DH_ERR_ARG;
        if ((uintptr_t)grads[k] % (dtype == DH_F32 ? 4 : 2)) return DH_ERR_ALIGN;
    }
    const int64_t need = dh_grad_parts(n, count);
    if (parts < need) return DH_ERR_WORKSPACE;
    if (need && (!partial || (uintptr_t)partial % 8)) return DH_ERR_ARG;
    hipStream_t st = (hipStream_t)stream;
    for (int lo = 0; lo < count; lo += READ) {
        Table<false> t;
        const int chunks = fill(&t, grads, nullptr, n, lo, count);
        if (chunks == 0) continue;
        const int groups = groups_of(chunks);
        if (dtype == DH_F32) launch_power<float>(t, norm, groups, partial, st);
        else if (dtype == DH_F16) launch_power<_Float16>(t, norm, groups, partial, st);
        else launch_power<__bf16>(t, norm, groups, partial, st);
        partial += groups;
    }
    return dh_launch_status();
}

extern "C" int dh_grad_norm(const double* partial, int64_t parts, int norm, const float* scale, double* sum, float* out, void* stream)
{
    if (parts < 0 || parts >= (1ll << 31) || (parts && !partial) || !kinds(norm) || (!sum && !out)) return DH_ERR_ARG;
    hipStream_t st = (hipStream_t)stream;
    if (norm == DH_NORM_1) hipLaunchKernelGGL((k_grad_join<DH_NORM_1>), dim3(1), dim3(256), 0, st, partial, (int)parts, scale, sum, out);
    else if (norm == DH_NORM_2) hipLaunchKernelGGL((k_grad_join<DH_NORM_2>), dim3(1), dim3(256), 0, st, partial, (int)parts, scale, sum, out);
    else hipLaunchKernelGGL((k_grad_join<DH_NORM_MAX>), dim3(1), dim3(256), 0, st, partial, (int)parts, scale, sum, out);
    return dh_launch_status();
}

extern "C" int dh_grad_clip(const void* const* grads, void* const* out, const int64_t* n, int count, int dtype, int out_dtype, int norm,
                            const double* partial, int64_t parts, const float* scale, double max_norm, float* norm_out, void* stream)
{
    if (!sized(n, count) || (count && (!grads || !out)) || !types(dtype) || (out_dtype != dtype && out_dtype != DH_F32) || !kinds(norm))
        return DH_ERR_ARG;
    if (parts < 0 || parts >= (1ll << 31) || (parts && !partial) || !(max_norm >= 0.0)) return DH_ERR_ARG;
    for (int k = 0; k < count; ++k) {
        if (n[k] && (!grads[k] || !out[k])) return DH_ERR_ARG;
        if ((uintptr_t)grads[k] % (dtype == DH_F32 ? 4 : 2) || (uintptr_t)out[k] % (out_dtype == DH_F32 ? 4 : 2)) return DH_ERR_ALIGN;
    }
    hipStream_t st = (hipStream_t)stream;
    const bool in_place = out_dtype == dtype && std::equal(grads, grads + count, out);
    const bool told = in_place ? clip_all<false>(grads, out, n, count, dtype, out_dtype, norm, partial, (int)parts, scale, max_norm, norm_out, st)
                               : clip_all<true>(grads, out, n, count, dtype, out_dtype, norm, partial, (int)parts, scale, max_norm, norm_out, st);
    if (!told && norm_out) return dh_grad_norm(partial, parts, norm, scale, nullptr, norm_out, stream);      // nothing to scale
    return dh_launch_status();
}
