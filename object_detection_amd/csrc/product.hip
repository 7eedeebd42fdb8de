// Matrix products C(i,j) = sum_r A(i,r) B(j,r) on the matrix cores, with the bias, the activation and the residual applied to
// the accumulators before the one rounding of the result; and the two operators around their backward pass.
//
// One kernel serves the forward pass and both gradients, for row-major tokens and for channel-major maps, because in each of
// them an operand is either contiguous along the reduction ("R", a row of W or of tokens) or along its own index ("C"):
//
//               forward                     gradient of the input        gradient of the weight
//   tokens      A = x   R, B = W   R        A = dz  R, B = W^T C         A = dz^T C, B = x^T  C   (reduction over the tokens)
//   maps        A = W   R, B = x_b C        A = W^T C, B = dz_b C        A = dz_b R, B = x_b  R   (reduction over b and cells)
#include "../../include/dethead.h"
#include "dh_common.h"
#include <hip/hip_fp16.h>
#include <hip/hip_bf16.h>
#include <math.h>

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef unsigned int u4 __attribute__((ext_vector_type(4)));

// ---- element types: conversions, and how many elements one 16-byte chunk holds ----
template <typename T> struct Elem;
template <> struct Elem<float> {
    static constexpr int CH = 4;
    __device__ static float up(float v) { return v; }
    __device__ static float down(float v) { return v; }
};
template <> struct Elem<_Float16> {
    static constexpr int CH = 8;
    __device__ static float up(_Float16 v) { return (float)v; }
    __device__ static _Float16 down(float v) { return (_Float16)v; }
};
template <> struct Elem<__bf16> {
    static constexpr int CH = 8;
    __device__ static float up(__bf16 v) { return (float)v; }
    __device__ static __bf16 down(float v) { return (__bf16)v; }
};

__device__ __forceinline__ float act_value(float z, int act)
{
    switch (act) {
    case DH_ACT_RELU: return z > 0.f ? z : (z != z ? z : 0.f);      // a NaN stays one
    case DH_ACT_SILU: return z / (1.f + expf(-z));
    case DH_ACT_SIGMOID: return 1.f / (1.f + expf(-z));
    case DH_ACT_GELU: return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
    default: return z;
    }
}

__device__ __forceinline__ float act_slope(float z, int act)
{
    switch (act) {
    case DH_ACT_RELU: return z > 0.f ? 1.f : 0.f;
    case DH_ACT_SILU: { const float s = 1.f / (1.f + expf(-z)); return s * (1.f + z * (1.f - s)); }
    case DH_ACT_SIGMOID: { const float s = 1.f / (1.f + expf(-z)); return s * (1.f - s); }
    case DH_ACT_GELU:
        return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * 0.39894228040143268f * expf(-0.5f * z * z);
    default: return 1.f;
    }
}

struct Plan {               // one problem of a launch and how it is cut
    dh_product p;
    int tiles_i, tiles_j;   // output tiles
    int steps;              // reduction steps of one output tile (all batches when the batch is reduced)
    int batch_steps;        // reduction steps of one batch
    int split, per;         // workgroups along the reduction, and steps of each
    int out_batches;        // batches of the output (1 when the batch is reduced)
    int first;              // first workgroup of this problem
    int vec_out;            // rows of out / z / residual can be accessed in 16-byte pieces
    float* partial;         // split > 1: [split][out_batches][I][J]
};

struct Launch {
    Plan plan[DH_MAX_PRODUCTS];
    int n, total, act;
};

// 16 bytes of an operand that is contiguous along the direction of `at` (extent `end`); elements beyond it are zero.
template <typename T, bool VEC>
__device__ __forceinline__ u4 load_chunk(const T* __restrict__ row, int at, int end)
{
    constexpr int CH = Elem<T>::CH;
    u4 v = {0, 0, 0, 0};
    if (VEC) {                                  // aligned, and the extent is a multiple of the chunk
        if (at < end) v = *reinterpret_cast<const u4*>(row + at);
    } else if (at + CH <= end) {
        __builtin_memcpy(&v, row + at, 16);     // any alignment of the element type
    } else {
        T e[CH];
        __builtin_memset(e, 0, 16);
#pragma unroll
        for (int k = 0; k < CH; ++k)
            if (at + k < end) e[k] = row[at + k];
        __builtin_memcpy(&v, e, 16);
    }
    return v;
}

// An operand's tile in LDS.  X: rows of the tile along the operand's own index, BR: along the reduction.
//   R (contiguous along the reduction): [X][BR], one row is 128 bytes = 8 chunks; chunk c of row x sits at c ^ key(x), so that
//     the 16 rows a fragment read touches spread over all banks.
//   C (contiguous along its own index): [BR][X]; chunk c of row r sits at c ^ key(r).  The 16-bit types read their fragments
//     with the transposing LDS read (a lane receives four values of its column from four rows), fp32 reads single words.
// PAIR: the order of the operand's indices inside a wave's tile.  The B operand of a 16-bit product takes
//   j = 32 (t/2) + 8 (m/4) + 4 (t%2) + m%4 for value m of fragment t, so that a lane's accumulators of two fragments are eight
//   consecutive values of C's row = one 16-byte store; the others take j = 16 t + m.
template <typename T, int X, int BR, bool RC, bool PAIR>
struct Tile {
    static constexpr int CH = Elem<T>::CH;
    static constexpr int CHUNKS = X * BR / CH;
    static constexpr int ROW_CHUNKS = (RC ? BR : X) / CH;

    __device__ static int key(int row)
    {
        if (RC) return PAIR ? ((row & 3) | ((row >> 1) & 4)) : (row & 7);
        if (sizeof(T) == 4) return (((row >> 2) & 3) * 4) & (ROW_CHUNKS - 1);
        return ((row & 3) * (PAIR ? 4 : 2)) & (ROW_CHUNKS - 1);
    }

    // chunk number k of the tile in memory order
    template <bool VEC>
    __device__ static u4 fetch(const T* __restrict__ base, int64_t ld, int x0, int xend, int r0, int rend, int k)
    {
        const int row = k / ROW_CHUNKS, c = k % ROW_CHUNKS;
        if (RC) {
            const int x = x0 + row < xend ? x0 + row : xend - 1;      // rows behind the end repeat the last: never stored
            return load_chunk<T, VEC>(base + (int64_t)x * ld, r0 + c * CH, rend);
        }
        u4 zero = {0, 0, 0, 0};
        if (r0 + row >= rend) return zero;
        return load_chunk<T, VEC>(base + (int64_t)(r0 + row) * ld, x0 + c * CH, xend);
    }

    __device__ static void store(T* lds, int k, u4 v)
    {
        const int row = k / ROW_CHUNKS, c = k % ROW_CHUNKS;
        *reinterpret_cast<u4*>(lds + (row * ROW_CHUNKS + (c ^ key(row))) * CH) = v;
    }

    // the tile-local index of value m of fragment t
    __device__ static int index(int t, int m) { return PAIR ? 32 * (t >> 1) + 8 * (m >> 2) + 4 * (t & 1) + (m & 3) : 16 * t + m; }

    // 16-bit types: 8 reduction values (32 kk + 8 (lane/16) ..) of fragment t, the wave's tile starting at x0
    __device__ static s8 frag16(const T* lds, int x0, int t, int kk, int lane)
    {
        const int m = lane & 15, g = lane >> 4;
        if (RC) {
            const int x = x0 + index(t, m);
            return *reinterpret_cast<const s8*>(lds + (x * ROW_CHUNKS + ((4 * kk + g) ^ key(x))) * CH);
        }
        const int x = x0 + index(t, 4 * (m & 3));          // four consecutive columns that this lane reads for its group
        s8 v;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = 32 * kk + 8 * g + 4 * h + (m >> 2);
            const T* at = lds + (r * ROW_CHUNKS + ((x / CH) ^ key(r))) * CH + (x & (CH - 1));
            const s4 q = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s4*)(reinterpret_cast<s4*>(const_cast<T*>(at))));
            v[4 * h] = q[0]; v[4 * h + 1] = q[1]; v[4 * h + 2] = q[2]; v[4 * h + 3] = q[3];
        }
        return v;
    }

    // fp32: 4 reduction values 16 kk + 4 (lane/16) + e of fragment t
    __device__ static f4 frag32(const T* lds, int x0, int t, int kk, int lane)
    {
        const int m = lane & 15, g = lane >> 4;
        const int x = x0 + index(t, m);
        if (RC) return *reinterpret_cast<const f4*>(lds + (x * ROW_CHUNKS + ((4 * kk + g) ^ key(x))) * CH);
        f4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = 16 * kk + 4 * g + e;
            v[e] = ((const float*)lds)[(r * ROW_CHUNKS + ((x / CH) ^ key(r))) * CH + (x & 3)];
        }
        return v;
    }
};

// Two reads of 32 reduction values each for the 16-bit types, 16 values of four single-value instructions for fp32.
template <typename T> __device__ __forceinline__ f4 mma16(s8 a, s8 b, f4 c);
template <> __device__ __forceinline__ f4 mma16<_Float16>(s8 a, s8 b, f4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f4 mma16<__bf16>(s8 a, s8 b, f4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

// The last step on N consecutive values of a row of C: bias, activation, residual, rounding.
template <typename T, int N>
__device__ __forceinline__ void finish(const dh_product& p, int act, bool vec, int b, int i, int j, int J, const float* acc)
{
    const int64_t o = (int64_t)b * p.o_batch + (int64_t)i * p.ldo + j;
    const int64_t ro = (int64_t)b * p.res_batch + (int64_t)i * p.ldr + j;
    const T* bias = (const T*)p.bias;
    const T* res = (const T*)p.residual;
    const int n = J - j < N ? J - j : N;
    const bool whole = vec && n == N;
    alignas(16) T zs[N], ys[N], rs[N];
    if (res) {
        if (whole) __builtin_memcpy(rs, __builtin_assume_aligned(res + ro, N * sizeof(T) < 16 ? N * sizeof(T) : 16), sizeof(rs));
        else
#pragma unroll
            for (int k = 0; k < N; ++k) rs[k] = k < n ? res[ro + k] : T(0);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
        float z = acc[k];
        if (bias) z += p.bias_on_i ? Elem<T>::up(bias[i]) : (k < n ? Elem<T>::up(bias[j + k]) : 0.f);
        zs[k] = Elem<T>::down(z);
        float y = act_value(z, act);
        if (res) y += Elem<T>::up(rs[k]);
        ys[k] = Elem<T>::down(y);
    }
    T* out = (T*)p.out + o;
    T* zout = p.z ? (T*)p.z + o : nullptr;
    if (whole) {
        __builtin_memcpy(__builtin_assume_aligned(out, N * sizeof(T) < 16 ? N * sizeof(T) : 16), ys, sizeof(ys));
        if (zout) __builtin_memcpy(__builtin_assume_aligned(zout, N * sizeof(T) < 16 ? N * sizeof(T) : 16), zs, sizeof(zs));
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (k < n) { out[k] = ys[k]; if (zout) zout[k] = zs[k]; }
    }
}

template <typename T, int BI, int BJ, int WI, int WJ, bool ARC, bool BRC, bool VEC>
__global__ void __launch_bounds__(WI * WJ * 64) k_product(const Launch L)
{
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int BR = F32 ? 32 : 64;
    constexpr int THREADS = WI * WJ * 64;
    constexpr int TI = BI / WI / 16, TJ = BJ / WJ / 16;
    constexpr bool PAIR = !F32;
    typedef Tile<T, BI, BR, ARC, false> TA;
    typedef Tile<T, BJ, BR, BRC, PAIR> TB;
    constexpr int NA = TA::CHUNKS / THREADS, NB = TB::CHUNKS / THREADS;
    static_assert(TA::CHUNKS % THREADS == 0 && TB::CHUNKS % THREADS == 0, "whole chunks per thread");
    static_assert(!PAIR || TJ % 2 == 0, "fragments of B go in pairs");
    __shared__ __align__(16) T lds_a[2][BI * BR];
    __shared__ __align__(16) T lds_b[2][BJ * BR];

    // consecutive workgroup numbers go to the 8 XCDs in turn: each XCD takes a contiguous eighth of the tiles, so that tiles
    // which share an operand meet in one L2
    const int per_xcd = (L.total + 7) / 8;
    int tile = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
    if (tile >= L.total) return;
    int w = 0;
    while (w + 1 < L.n && tile >= L.plan[w + 1].first) ++w;
    const Plan& q = L.plan[w];
    const dh_product& p = q.p;
    tile -= q.first;
    const int ti = tile % q.tiles_i; tile /= q.tiles_i;
    const int tj = tile % q.tiles_j; tile /= q.tiles_j;
    const int ob = tile % q.out_batches;
    const int s = tile / q.out_batches;
    const int i0 = ti * BI, j0 = tj * BJ;
    const int k_begin = s * q.per, k_end = k_begin + q.per < q.steps ? k_begin + q.per : q.steps;

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wi = (wave / WJ) * (BI / WI), wj = (wave % WJ) * (BJ / WJ);
    u4 ra[NA], rb[NB];
    f4 acc[TI][TJ];
#pragma unroll
    for (int a = 0; a < TI; ++a)
#pragma unroll
        for (int b = 0; b < TJ; ++b) acc[a][b] = f4{0.f, 0.f, 0.f, 0.f};

    auto fetch = [&](int k) {
        const int b = p.reduce_batch ? k / q.batch_steps : ob;
        const int r0 = (p.reduce_batch ? k - b * q.batch_steps : k) * BR;
        const T* A = (const T*)p.a + (int64_t)b * p.a_batch;
        const T* B = (const T*)p.b + (int64_t)b * p.b_batch;
#pragma unroll
        for (int c = 0; c < NA; ++c) ra[c] = TA::template fetch<VEC>(A, p.lda, i0, p.I, r0, p.R, c * THREADS + tid);
#pragma unroll
        for (int c = 0; c < NB; ++c) rb[c] = TB::template fetch<VEC>(B, p.ldb, j0, p.J, r0, p.R, c * THREADS + tid);
    };
    auto stage = [&](int at) {
#pragma unroll
        for (int c = 0; c < NA; ++c) TA::store(lds_a[at], c * THREADS + tid, ra[c]);
#pragma unroll
        for (int c = 0; c < NB; ++c) TB::store(lds_b[at], c * THREADS + tid, rb[c]);
    };

    if (k_begin < k_end) { fetch(k_begin); stage(0); }
    __syncthreads();
    int at = 0;
    for (int k = k_begin; k < k_end; ++k) {
        if (k + 1 < k_end) fetch(k + 1);
        if constexpr (F32) {
#pragma unroll
            for (int kk = 0; kk < BR / 16; ++kk) {
                f4 fa[TI], fb[TJ];
#pragma unroll
                for (int a = 0; a < TI; ++a) fa[a] = TA::frag32(lds_a[at], wi, a, kk, lane);
#pragma unroll
                for (int b = 0; b < TJ; ++b) fb[b] = TB::frag32(lds_b[at], wj, b, kk, lane);
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int a = 0; a < TI; ++a)
#pragma unroll
                        for (int b = 0; b < TJ; ++b)
                            acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[b][e], fa[a][e], acc[a][b], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int kk = 0; kk < BR / 32; ++kk) {
                s8 fa[TI], fb[TJ];
#pragma unroll
                for (int a = 0; a < TI; ++a) fa[a] = TA::frag16(lds_a[at], wi, a, kk, lane);
#pragma unroll
                for (int b = 0; b < TJ; ++b) fb[b] = TB::frag16(lds_b[at], wj, b, kk, lane);
#pragma unroll
                for (int a = 0; a < TI; ++a)
#pragma unroll
                    for (int b = 0; b < TJ; ++b) acc[a][b] = mma16<T>(fb[b], fa[a], acc[a][b]);
            }
        }
        if (k + 1 < k_end) stage(at ^ 1);
        __syncthreads();
        at ^= 1;
    }

    // C's row i is the lane's column of the accumulator, its four values are consecutive in j (twice that for a pair)
    constexpr int G = PAIR ? 2 : 1;
#pragma unroll
    for (int a = 0; a < TI; ++a) {
        const int i = i0 + wi + 16 * a + (lane & 15);
#pragma unroll
        for (int b = 0; b < TJ; b += G) {
            const int j = j0 + wj + TB::index(b, 4 * (lane >> 4));
            if (i >= p.I || j >= p.J) continue;
            float v[4 * G];
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * g + e] = acc[a][b + g][e];
            if (q.split > 1) {
                float* o = q.partial + (((int64_t)s * q.out_batches + ob) * p.I + i) * p.J + j;
#pragma unroll
                for (int e = 0; e < 4 * G; ++e)
                    if (j + e < p.J) o[e] = v[e];
            } else {
                finish<T, 4 * G>(p, L.act, q.vec_out != 0, ob, i, j, p.J, v);
            }
        }
    }
}

// Sums the partial products of the workgroups along the reduction, in their order, and finishes them.
template <typename T>
__global__ void __launch_bounds__(256) k_product_join(const Plan q, int act)
{
    const dh_product& p = q.p;
    const int64_t n = (int64_t)q.out_batches * p.I * p.J;
    for (int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x; k < n; k += (int64_t)gridDim.x * 256) {
        float v = 0.f;
        for (int s = 0; s < q.split; ++s) v += q.partial[(int64_t)s * n + k];
        const int j = (int)(k % p.J);
        const int64_t rest = k / p.J;
        finish<T, 1>(p, act, false, (int)(rest / p.I), (int)(rest % p.I), j, p.J, &v);
    }
}

constexpr int TILE = 128, SMALL = 64;

int cut(const dh_product* ps, int n, int dtype, Launch* L, float* ws, size_t* ws_bytes, bool* vec, int* tile)
{
    const int64_t ch = dtype == DH_F32 ? 4 : 8, br = dtype == DH_F32 ? 32 : 64;
    const int cus = 256;
    int64_t large = 0;
    for (int w = 0; w < n; ++w)
        large += (int64_t)((ps[w].I + TILE - 1) / TILE) * ((ps[w].J + TILE - 1) / TILE) * (ps[w].reduce_batch ? 1 : ps[w].batch);
    const int t = large >= cus ? TILE : SMALL;
    *tile = t;
    *vec = true;
    int64_t total = 0;
    size_t bytes = 0;
    for (int w = 0; w < n; ++w) {
        const dh_product& p = ps[w];
        Plan& q = L->plan[w];
        q.p = p;
        q.tiles_i = (p.I + t - 1) / t;
        q.tiles_j = (p.J + t - 1) / t;
        q.batch_steps = (int)((p.R + br - 1) / br);
        const int64_t steps = (int64_t)q.batch_steps * (p.reduce_batch ? p.batch : 1);
        q.out_batches = p.reduce_batch ? 1 : p.batch;
        const int64_t tiles = (int64_t)q.tiles_i * q.tiles_j * q.out_batches;
        if (steps >= (1ll << 31) || tiles >= (1ll << 28)) return DH_ERR_ARG;
        q.steps = (int)steps;
        int64_t split = tiles >= 2 * cus || tiles == 0 ? 1 : (2 * cus + tiles - 1) / tiles;
        if (split > steps / 4) split = steps / 4;           // at least four steps each
        if (split < 1) split = 1;
        q.per = (int)((steps + split - 1) / split);
        q.split = q.per ? (int)((steps + q.per - 1) / q.per) : 1;
        q.partial = nullptr;
        if (q.split > 1) {
            q.partial = (float*)((char*)ws + bytes);
            bytes += ((size_t)q.split * q.out_batches * p.I * p.J * sizeof(float) + 255) & ~(size_t)255;
        }
        q.first = (int)total;
        total += tiles * q.split;
        if (total >= (1ll << 30)) return DH_ERR_ARG;
        const int64_t all = p.lda | p.ldb | p.a_batch | p.b_batch;
        const int64_t ea = p.a_by_reduction ? p.R : p.I, eb = p.b_by_reduction ? p.R : p.J;
        if (all % ch || ea % ch || eb % ch || !dh_aligned16(p.a) || !dh_aligned16(p.b)) *vec = false;
        q.vec_out = p.ldo % ch == 0 && p.o_batch % ch == 0 && dh_aligned16(p.out) && (!p.z || dh_aligned16(p.z)) &&
                    (!p.residual || (p.ldr % ch == 0 && p.res_batch % ch == 0 && dh_aligned16(p.residual)));
    }
    L->n = n;
    L->total = (int)total;
    *ws_bytes = bytes;
    return DH_OK;
}

template <typename T, int B, bool ARC, bool BRC>
void launch_tile(const Launch& L, bool vec, hipStream_t st)
{
    const dim3 grid((unsigned)((L.total + 7) / 8 * 8));
    if (vec) hipLaunchKernelGGL((k_product<T, B, B, 2, 2, ARC, BRC, true>), grid, dim3(256), 0, st, L);
    else hipLaunchKernelGGL((k_product<T, B, B, 2, 2, ARC, BRC, false>), grid, dim3(256), 0, st, L);
}

template <typename T>
int launch(const Launch& L, bool arc, bool brc, bool vec, int tile, hipStream_t st)
{
    if (L.total > 0) {
        if (tile == TILE) {
            if (arc && brc) launch_tile<T, TILE, true, true>(L, vec, st);
            else if (arc) launch_tile<T, TILE, true, false>(L, vec, st);
            else launch_tile<T, TILE, false, false>(L, vec, st);
        } else {
            if (arc && brc) launch_tile<T, SMALL, true, true>(L, vec, st);
            else if (arc) launch_tile<T, SMALL, true, false>(L, vec, st);
            else launch_tile<T, SMALL, false, false>(L, vec, st);
        }
    }
    for (int w = 0; w < L.n; ++w)
        if (L.plan[w].split > 1) {
            const int64_t n = (int64_t)L.plan[w].out_batches * L.plan[w].p.I * L.plan[w].p.J;
            const int64_t blocks = (n + 255) / 256;
            hipLaunchKernelGGL((k_product_join<T>), dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, st, L.plan[w], L.act);
        }
    return dh_launch_status();
}

int check(const dh_product* ps, int n, int dtype, int activation)
{
    if (!ps || n < 1 || n > DH_MAX_PRODUCTS || dtype < DH_F32 || dtype > DH_BF16 || activation < 0 || activation > DH_ACT_LAST)
        return DH_ERR_ARG;
    const uintptr_t esize = dtype == DH_F32 ? 4 : 2;
    for (int w = 0; w < n; ++w) {
        const dh_product& p = ps[w];
        if (p.I < 0 || p.J < 0 || p.R < 0 || p.batch < 0 || p.lda < 0 || p.ldb < 0 || p.ldo < 0 || p.ldr < 0) return DH_ERR_ARG;
        if (!!p.a_by_reduction != !!ps[0].a_by_reduction || !!p.b_by_reduction != !!ps[0].b_by_reduction) return DH_ERR_ARG;
        if (!p.a_by_reduction && p.b_by_reduction) return DH_ERR_ARG;      // no caller has that pair
        const bool work = p.I > 0 && p.J > 0 && (p.reduce_batch || p.batch > 0);
        if (work && !p.out) return DH_ERR_ARG;
        if (work && p.R > 0 && p.batch > 0 && (!p.a || !p.b)) return DH_ERR_ARG;
        const uintptr_t all = (uintptr_t)p.a | (uintptr_t)p.b | (uintptr_t)p.out | (uintptr_t)p.z | (uintptr_t)p.residual | (uintptr_t)p.bias;
        if (all % esize) return DH_ERR_ALIGN;
    }
    return DH_OK;
}

// ---- dz = dy * act'(z) and the bias gradient ----
// dy is [outer][n][inner]; the bias gradient sums over outer and inner.  SPLIT workgroups share one n (inner > 1) or one
// column block (inner == 1); their sums go to the workspace and are added in order by k_bias_join.
constexpr int BIAS_SPLIT = 64;

template <typename T>
__global__ void __launch_bounds__(256) k_slope_planes(const T* __restrict__ dy, const T* __restrict__ z, T* __restrict__ dz,
                                                      float* __restrict__ partial, int64_t outer, int64_t n, int64_t inner, int act)
{
    const int64_t c = blockIdx.x / BIAS_SPLIT, s = blockIdx.x % BIAS_SPLIT;
    float sum = 0.f;
    for (int64_t o = s; o < outer; o += BIAS_SPLIT) {
        const int64_t at = (o * n + c) * inner;
        for (int64_t k = threadIdx.x; k < inner; k += 256) {
            float g = Elem<T>::up(dy[at + k]);
            if (z) { g *= act_slope(Elem<T>::up(z[at + k]), act); dz[at + k] = Elem<T>::down(g); }
            sum += g;
        }
    }
    if (!partial) return;
    __shared__ float sums[4];
    sum = dh_wave_sum(sum);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) partial[s * n + c] = sums[0] + sums[1] + sums[2] + sums[3];
}

template <typename T>
__global__ void __launch_bounds__(256) k_slope_rows(const T* __restrict__ dy, const T* __restrict__ z, T* __restrict__ dz,
                                                    float* __restrict__ partial, int64_t rows, int64_t n, int act)
{
    const int64_t c = (blockIdx.x / BIAS_SPLIT) * 64 + (threadIdx.x & 63), s = blockIdx.x % BIAS_SPLIT;
    float sum = 0.f;
    if (c < n)
        for (int64_t r = s * 4 + (threadIdx.x >> 6); r < rows; r += 4 * BIAS_SPLIT) {
            float g = Elem<T>::up(dy[r * n + c]);
            if (z) { g *= act_slope(Elem<T>::up(z[r * n + c]), act); dz[r * n + c] = Elem<T>::down(g); }
            sum += g;
        }
    if (!partial) return;
    __shared__ float sums[256];
    sums[threadIdx.x] = sum;
    __syncthreads();
    if (threadIdx.x < 64 && c < n)
        partial[s * n + c] = sums[threadIdx.x] + sums[threadIdx.x + 64] + sums[threadIdx.x + 128] + sums[threadIdx.x + 192];
}

template <typename T>
__global__ void __launch_bounds__(256) k_bias_join(const float* __restrict__ partial, T* __restrict__ dbias, int64_t n)
{
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= n) return;
    float sum = 0.f;
    for (int s = 0; s < BIAS_SPLIT; ++s) sum += partial[s * n + c];
    dbias[c] = Elem<T>::down(sum);
}

template <typename T>
int launch_slope(const void* dy, const void* z, void* dz, void* dbias, int64_t outer, int64_t n, int64_t inner, int act,
                 float* ws, hipStream_t st)
{
    float* partial = dbias ? ws : nullptr;
    if (inner > 1)
        hipLaunchKernelGGL((k_slope_planes<T>), dim3((unsigned)(n * BIAS_SPLIT)), dim3(256), 0, st, (const T*)dy, (const T*)z, (T*)dz,
                           partial, outer, n, inner, act);
    else
        hipLaunchKernelGGL((k_slope_rows<T>), dim3((unsigned)((n + 63) / 64 * BIAS_SPLIT)), dim3(256), 0, st, (const T*)dy, (const T*)z,
                           (T*)dz, partial, outer, n, act);
    if (dbias)
        hipLaunchKernelGGL((k_bias_join<T>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, partial, (T*)dbias, n);
    return dh_launch_status();
}

}  // namespace

extern "C" size_t dh_products_workspace(const dh_product* products, int n, int dtype)
{
    if (check(products, n, dtype, 0) != DH_OK) return 0;
    Launch L;
    size_t bytes = 0;
    bool vec;
    int tile;
    return cut(products, n, dtype, &L, nullptr, &bytes, &vec, &tile) == DH_OK ? bytes : 0;
}

extern "C" int dh_products(const dh_product* products, int n, int dtype, int activation, void* workspace, size_t workspace_bytes,
                           void* stream)
{
    int rc = check(products, n, dtype, activation);
    if (rc != DH_OK) return rc;
    Launch L;
    size_t bytes = 0;
    bool vec;
    int tile;
    rc = cut(products, n, dtype, &L, (float*)workspace, &bytes, &vec, &tile);
    if (rc != DH_OK) return rc;
    if (bytes > workspace_bytes || (bytes && !workspace)) return DH_ERR_WORKSPACE;
    if (bytes && !dh_aligned16(workspace)) return DH_ERR_ALIGN;
    L.act = activation;
    const bool arc = products[0].a_by_reduction != 0, brc = products[0].b_by_reduction != 0;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == DH_F32) return launch<float>(L, arc, brc, vec, tile, st);
    if (dtype == DH_F16) return launch<_Float16>(L, arc, brc, vec, tile, st);
    return launch<__bf16>(L, arc, brc, vec, tile, st);
}

extern "C" size_t dh_product_slope_workspace(int64_t n) { return n > 0 ? (size_t)n * BIAS_SPLIT * sizeof(float) : 0; }

extern "C" int dh_product_slope(const void* dy, const void* z, void* dz, void* dbias, int64_t outer, int64_t n, int64_t inner,
                                int activation, int dtype, void* workspace, size_t workspace_bytes, void* stream)
{
    if (outer < 0 || n < 0 || inner < 0 || dtype < DH_F32 || dtype > DH_BF16 || activation < 0 || activation > DH_ACT_LAST) return DH_ERR_ARG;
    if (n == 0 || (!z && !dbias)) return DH_OK;
    if (n >= (1ll << 24) || outer >= (1ll << 40) || inner >= (1ll << 40)) return DH_ERR_ARG;
    if (outer * inner > 0 && (!dy || (z && !dz))) return DH_ERR_ARG;
    if (dbias && (!workspace || workspace_bytes < dh_product_slope_workspace(n))) return DH_ERR_WORKSPACE;
    if (dbias && !dh_aligned16(workspace)) return DH_ERR_ALIGN;
    hipStream_t st = (hipStream_t)stream;
    float* ws = (float*)workspace;
    if (dtype == DH_F32) return launch_slope<float>(dy, z, dz, dbias, outer, n, inner, activation, ws, st);
    if (dtype == DH_F16) return launch_slope<_Float16>(dy, z, dz, dbias, outer, n, inner, activation, ws, st);
    return launch_slope<__bf16>(dy, z, dz, dbias, outer, n, inner, activation, ws, st);
}
