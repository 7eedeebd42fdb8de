// Matrix products C(i,j) = sum_r A(i,r) B(j,r) on the matrix cores, with the bias, the activation and the residual applied to
// the accumulators before the one rounding of the result; and the two operators around their backward pass.
//
// One kernel serves the forward pass and both gradients, for row-major tokens and for channel-major maps, because in each of
// them an operand is either contiguous along the reduction ("R", a row of W or of tokens) or along its own index ("C"):
//
//               forward                     gradient of the input        gradient of the weight
//   tokens      A = x   R, B = W   R        A = dz  R, B = W^T C         A = dz^T C, B = x^T  C   (reduction over the tokens)
//   maps        A = W   R, B = x_b C        A = W^T C, B = dz_b C        A = dz_b R, B = x_b  R   (reduction over b and cells)
#pragma once
#include "../../include/dethead.h"
#include "dh_common.h"
#include <hip/hip_fp16.h>
#include <hip/hip_bf16.h>
#include <math.h>
#include <type_traits>

namespace dhp {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef unsigned int u4 __attribute__((ext_vector_type(4)));
typedef unsigned int u2 __attribute__((ext_vector_type(2)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));

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

// Activations and their derivatives.  FAST (results that are rounded to 16 bits): exp2 and the reciprocal from the hardware
// (1 ulp each; what leaves fp32's normal range becomes zero, so a silu below 1e-36 does), and the normal distribution function from
// its tail, exp(-x^2) t (a1 + .. + a6 t^5) with t = 1 / (1 + 0.415 x): the form of Abramowitz & Stegun 7.1.26 with one term more, its
// coefficients found by linear programming so that the error stays below 2^-23 and, where that is more, below 2^-14 of the tail (an
// eighth of half an fp16 step; 7.1.26 itself is off by 1.6e-3 at -5 and 4e-2 at -14).  A gelu is 15 instructions instead of the
// library's 45, which at 8192 x 4096 outputs is 30 us of vector work.  fp32 results take (1 + erf) / 2, as the plain form does: its error
// of 2^-24 is of 1, not of the tail.
template <int ACT, bool FAST> struct Act;
template <bool FAST> struct Act<DH_ACT_NONE, FAST> {
    __device__ static float value(float z) { return z; }
    __device__ static float slope(float) { return 1.f; }
};
template <bool FAST> struct Act<DH_ACT_RELU, FAST> {
    __device__ static float value(float z) { return z > 0.f ? z : (z != z ? z : 0.f); }      // a NaN stays one
};
template <bool FAST> __device__ __forceinline__ float logistic(float z)
{
    if (FAST) return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504088896f * z));
    return 1.f / (1.f + expf(-z));
}
template <bool FAST> struct Act<DH_ACT_SILU, FAST> {
    __device__ static float value(float z) { return FAST ? z * logistic<true>(z) : z / (1.f + expf(-z)); }
    __device__ static float slope(float z) { const float s = logistic<FAST>(z); return s * (1.f + z * (1.f - s)); }
};
template <bool FAST> struct Act<DH_ACT_SIGMOID, FAST> {
    __device__ static float value(float z) { return logistic<FAST>(z); }
    __device__ static float slope(float z) { const float s = logistic<FAST>(z); return s * (1.f - s); }
};
template <bool FAST> struct Act<DH_ACT_GELU, FAST> {
    // the normal distribution function at z; bell: exp(-z^2 / 2)
    __device__ static float normal(float z, float* bell)
    {
        if (!FAST) {
            *bell = expf(-0.5f * z * z);
            return 0.5f * (1.f + erff(z * 0.70710678118654752f));
        }
        const float x = fabsf(z) * 0.70710678118654752f;
        const float t = __builtin_amdgcn_rcpf(fmaf(0.415f, x, 1.f));
        *bell = __builtin_amdgcn_exp2f(-0.72134752044448f * z * z);
        float h = fmaf(-0.0851841997f, t, 0.260638247f);
        h = fmaf(h, t, -0.0644399153f);
        h = fmaf(h, t, 0.165055248f);
        h = fmaf(h, t, 0.10605487f);
        h = fmaf(h, t, 0.11787567f) * t * *bell;              // (1 - erf(x)) / 2
        return z > 0.f ? 1.f - h : h;
    }
    __device__ static float value(float z) { float bell; return z * normal(z, &bell); }
    __device__ static float slope(float z) { float bell; const float n = normal(z, &bell); return fmaf(z * 0.39894228040143268f, bell, n); }
};

// dy act'(z).  A relu passes dy on or stops it: an infinite dy where it stops is 0, and a NaN z passes, as in torch.
template <int ACT, bool FAST> __device__ __forceinline__ float act_back(float dy, float z)
{
    if constexpr (ACT == DH_ACT_RELU) return z <= 0.f ? 0.f : dy;
    else return dy * Act<ACT, FAST>::slope(z);
}

// f.template operator()<ACT>() for the activation of a launch
template <typename F> __device__ __forceinline__ void with_act(int act, F&& f)
{
    if (act == DH_ACT_NONE) f(std::integral_constant<int, DH_ACT_NONE>());
    else if (act == DH_ACT_RELU) f(std::integral_constant<int, DH_ACT_RELU>());
    else if (act == DH_ACT_SILU) f(std::integral_constant<int, DH_ACT_SILU>());
    else if (act == DH_ACT_GELU) f(std::integral_constant<int, DH_ACT_GELU>());
    else f(std::integral_constant<int, DH_ACT_SIGMOID>());
}

struct Plan {               // one problem of a launch and how it is cut
    dh_product p;
    int tiles_i, tiles_j;   // output tiles
    int steps;              // reduction steps of one output tile (all batches when the batch is reduced)
    int batch_steps;        // reduction steps of one batch
    int split, per;         // workgroups along the reduction, and steps of each
    int out_batches;        // batches of the output (1 when the batch is reduced)
    int count;              // workgroups of this problem
    dh_fastdiv by_plane, by_group, by_tail, by_batches;      // tiles_i tiles_j, 8 tiles_j, the last group's height, out_batches
    int stream;             // out and z are stored past the caches, in 16-byte pieces
    float* partial;         // split > 1: [split][out_batches][I][J]
    float* partial_sum;     // split > 1 and a_sum: [split][I]
};

struct Launch {
    int n, total, act;
    int first[DH_MAX_PRODUCTS];     // first workgroup of each problem (a multiple of 8)
    Plan plan[DH_MAX_PRODUCTS];
};

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
        if (RC && ROW_CHUNKS == 4) return PAIR ? (((row >> 1) & 1) | ((row >> 2) & 2)) : ((row >> 1) & 3);
        if (RC) return PAIR ? ((row & 3) | ((row >> 1) & 4)) : (row & 7);
        if (sizeof(T) == 4) return (((row >> 2) & 3) * 4) & (ROW_CHUNKS - 1);
        return ((row & 3) * (PAIR ? 4 : 2)) & (ROW_CHUNKS - 1);
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

// How an operand's tile comes from memory to LDS.
//
// Stream (everything aligned to 16 bytes): the copy goes from memory to LDS without passing through registers.  The hardware
// puts lane l's 16 bytes at M0 + 16 l, so the swizzle is applied to the address that each lane reads.  Offsets are set once; a
// reduction step only moves the scalar base.  The copies are written in assembly because the compiler, which cannot tell the
// ring's buffers apart, would wait for all of them before every fragment read; the kernel waits with vmcnt itself.
template <typename T, int X, int BR, bool RC, bool PAIR, int THREADS>
struct Stream {
    typedef Tile<T, X, BR, RC, PAIR> TL;
    static constexpr int CH = Elem<T>::CH, N = TL::CHUNKS / THREADS, ROWS = THREADS / TL::ROW_CHUNKS;
    static_assert(TL::CHUNKS % THREADS == 0 && THREADS % TL::ROW_CHUNKS == 0, "whole rows of chunks per pass");
    uint32_t offset[N];         // bytes from the tile's origin
    const char* base;           // the tile's origin at the current step
    int64_t step;               // bytes

    __device__ void begin(const T* operand, int64_t ld, int x0, int xend, int r0)
    {
        const int row = threadIdx.x / TL::ROW_CHUNKS, slot = threadIdx.x % TL::ROW_CHUNKS;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int y = row + k * ROWS, c = slot ^ TL::key(y);
            // what lies behind the operand's end repeats its last row or column: those sums are not stored
            const int64_t o = RC ? (int64_t)(x0 + y < xend ? y : xend - 1 - x0) * ld + c * CH
                                 : (int64_t)y * ld + (x0 + c * CH < xend ? c * CH : xend - CH - x0);
            offset[k] = (uint32_t)(o * (int64_t)sizeof(T));
        }
        base = (const char*)(operand + (RC ? (int64_t)x0 * ld + r0 : (int64_t)r0 * ld + x0));
        step = (RC ? BR : BR * ld) * (int64_t)sizeof(T);
    }

    // copies the step's chunks to `lds` (the wave's own first slot) and moves on; `left`: reduction values that remain
    __device__ void copy(T* lds, int left)
    {
        const uint32_t to = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) T*)lds);
        if (left >= BR) {
#pragma unroll
            for (int k = 0; k < N; ++k) one(to + k * THREADS * 16, offset[k]);
        } else {                // the end of the reduction: zeros behind it
            const int row = threadIdx.x / TL::ROW_CHUNKS, slot = threadIdx.x % TL::ROW_CHUNKS, lane = threadIdx.x & 63;
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const int y = row + k * ROWS, c = slot ^ TL::key(y);
                if (RC ? c * CH < left : y < left) one(to + k * THREADS * 16, offset[k]);
                else *reinterpret_cast<u4*>(lds + (k * THREADS + lane) * CH) = u4{0, 0, 0, 0};
            }
            asm volatile("s_waitcnt vmcnt(0)" : : : "memory");      // a wave may have skipped some: the count is not N
        }
        base += step;
    }

    __device__ void one(uint32_t to, uint32_t from) const
    {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(to), "v"(from), "s"(base) : "m0", "memory");
    }
};

// Waits until at most N of this wave's copies are on their way and its LDS reads are done, then for the other waves.
template <int N> __device__ __forceinline__ void wait_and_meet()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(N) : "memory");
}

// Feed (any alignment): through registers, one step ahead.
template <typename T, int X, int BR, bool RC, bool PAIR, int THREADS>
struct Feed {
    typedef T type;
    typedef Tile<T, X, BR, RC, PAIR> TL;
    static constexpr int CH = Elem<T>::CH, N = TL::CHUNKS / THREADS, ROWS = THREADS / TL::ROW_CHUNKS;
    static_assert(TL::CHUNKS % THREADS == 0 && THREADS % TL::ROW_CHUNKS == 0, "whole rows of chunks per thread");
    const T* at[N];
    const T* last;          // the last address from which a whole chunk can be read
    int64_t step;
    bool live;              // C: this thread's columns exist
    bool inside;            // the whole tile can be read
    int beyond;             // C at an edge: elements that one further row certainly has, up to a chunk

    __device__ static int tid() { return threadIdx.x & (THREADS - 1); }      // in the group of THREADS that shares a tile

    __device__ void begin(const T* base, int64_t ld, int x0, int xend, int r0, int rend)
    {
        const int row = tid() / TL::ROW_CHUNKS, c = tid() % TL::ROW_CHUNKS;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if (RC) {
                const int x = x0 + row + k * ROWS;
                at[k] = base + (int64_t)(x < xend ? x : xend - 1) * ld + r0 + c * CH;      // rows behind the end: never stored
            } else {
                // columns behind the end repeat the last ones: never stored
                const int x = x0 + c * CH < xend || xend < CH ? x0 + c * CH : xend - CH;
                at[k] = base + (int64_t)(r0 + row + k * ROWS) * ld + x;
            }
        }
        live = RC || x0 + c * CH < xend;
        // R: rows are clamped, so only the reduction can end.  C: a chunk over the end of a row reads on into the next one (columns
        // that are not stored), as long as 16 bytes of rows follow this step
        inside = RC || x0 + X <= xend;
        beyond = xend < CH ? 0 : (ld < CH ? (int)ld : CH);
        step = RC ? BR : BR * ld;
        last = base + (RC ? (int64_t)(xend - 1) * ld + rend : (int64_t)(rend - 1) * ld + xend) - CH;
    }

    // the chunks of a step of which `left` reduction values remain (BR or more: all); what lies behind them becomes zero
    __device__ void fetch(u4* v, int left)
    {
        const int after = left - BR < CH ? left - BR : CH;
        if (left >= BR && (inside || after * beyond >= CH)) {
#pragma unroll
            for (int k = 0; k < N; ++k) __builtin_memcpy(&v[k], at[k], 16);
        } else {
            const int row = tid() / TL::ROW_CHUNKS, c = tid() % TL::ROW_CHUNKS;
#pragma unroll
            for (int k = 0; k < N; ++k) {
                v[k] = u4{0, 0, 0, 0};
                const int have = RC ? left - c * CH : (live && row + k * ROWS < left ? CH : 0);    // elements of the chunk that count
                if (have >= CH && at[k] <= last) {
                    __builtin_memcpy(&v[k], at[k], 16);
                } else if (have > 0) {
                    T e[CH];
                    __builtin_memset(e, 0, 16);
#pragma unroll
                    for (int q = 0; q < CH; ++q)
                        if (q < have && at[k] + q < last + CH) e[q] = at[k][q];
                    __builtin_memcpy(&v[k], e, 16);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < N; ++k) at[k] += step;
    }

    __device__ static void stage(T* lds, const u4* v)
    {
#pragma unroll
        for (int k = 0; k < N; ++k) TL::store(lds, k * THREADS + tid(), v[k]);
    }
};

// One reduction step of a wave's tile from LDS.
// `sums`: also add up A's rows, as a product with ones.
template <typename T, typename TA, typename TB, int BR, int TI, int TJ>
__device__ __forceinline__ void multiply(f4 (&acc)[TI][TJ], f4 (&rows)[TI], bool sums, const T* la, const T* lb, int wi, int wj, int lane)
{
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int kk = 0; kk < BR / 16; ++kk) {
            f4 fa[TI], fb[TJ];
#pragma unroll
            for (int b = 0; b < TJ; ++b) fb[b] = TB::frag32(lb, wj, b, kk, lane);
#pragma unroll
            for (int a = 0; a < TI; ++a) fa[a] = TA::frag32(la, wi, a, kk, lane);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int a = 0; a < TI; ++a)
#pragma unroll
                    for (int b = 0; b < TJ; ++b)
                        acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[b][e], fa[a][e], acc[a][b], 0, 0, 0);
            if (sums) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int a = 0; a < TI; ++a) rows[a] = __builtin_amdgcn_mfma_f32_16x16x4f32(1.f, fa[a][e], rows[a], 0, 0, 0);
            }
        }
    } else {
        s8 ones;
#pragma unroll
        for (int e = 0; e < 8; ++e) ones[e] = std::is_same<T, __bf16>::value ? 0x3F80 : 0x3C00;
#pragma unroll
        for (int kk = 0; kk < BR / 32; ++kk) {
            s8 fa[TI], fb[TJ];
#pragma unroll
            for (int b = 0; b < TJ; ++b) fb[b] = TB::frag16(lb, wj, b, kk, lane);
#pragma unroll
            for (int a = 0; a < TI; ++a) fa[a] = TA::frag16(la, wi, a, kk, lane);
#pragma unroll
            for (int a = 0; a < TI; ++a)
#pragma unroll
                for (int b = 0; b < TJ; ++b) acc[a][b] = mma16<T>(fb[b], fa[a], acc[a][b]);
            if (sums) {
#pragma unroll
                for (int a = 0; a < TI; ++a) rows[a] = mma16<T>(ones, fa[a], rows[a]);
            }
        }
    }
}

// Which tile of which product a workgroup has.  Consecutive workgroup numbers go to the 8 XCDs in turn: each XCD takes a
// contiguous eighth of every product's tiles, in groups of 8 tiles along i that pass over j together, so that the tiles that run
// at one time on an XCD share their operands in its L2.
struct Place {
    int w, i0, j0, batch, s;
};
__device__ __forceinline__ bool place(const Launch& L, int BI, int BJ, Place* at)
{
    int w = 0;
#pragma unroll
    for (int k = 1; k < DH_MAX_PRODUCTS; ++k) w = k < L.n && (int)blockIdx.x >= L.first[k] ? k : w;
    const Plan& q = L.plan[w];
    const uint32_t local = blockIdx.x - L.first[w], per = (q.count + 7) / 8;
    uint32_t tile = (local & 7) * per + (local >> 3);
    if ((local >> 3) >= per || tile >= (uint32_t)q.count) return false;
    const uint32_t plane = q.tiles_i * q.tiles_j, rest = dh_div(tile, q.by_plane);
    tile -= rest * plane;
    const uint32_t group = dh_div(tile, q.by_group), in = tile - group * 8 * q.tiles_j;
    const uint32_t height = q.tiles_i - group * 8;
    const uint32_t tj = height >= 8 ? in >> 3 : dh_div(in, q.by_tail);
    at->w = w;
    at->i0 = (int)(group * 8 + in - tj * (height >= 8 ? 8 : height)) * BI;
    at->j0 = (int)tj * BJ;
    at->s = (int)dh_div(rest, q.by_batches);
    at->batch = (int)rest - at->s * q.out_batches;
    return true;
}

// The sums of A's rows that a wave holds (every lane of a column has the row's), to the result or to the partial sums.
template <typename T, int TI>
__device__ __forceinline__ void row_sums(const f4 (&rows)[TI], const Plan& q, const Place& at, int i0)
{
    const int lane = threadIdx.x & 63;
    if (lane >= 16) return;
#pragma unroll
    for (int a = 0; a < TI; ++a) {
        const int i = i0 + 16 * a + lane;
        if (i >= q.p.I) continue;
        if (q.split > 1) q.partial_sum[(int64_t)at.s * q.p.I + i] = rows[a][0];
        else ((T*)q.p.a_sum)[i] = Elem<T>::down(rows[a][0]);
    }
}

// What happens to a wave's accumulators.  They hold C in squares (a lane has four consecutive j of one row), memory wants rows:
// 16 rows at a time go through LDS (`mine`: 16 x W floats that only this wave uses), after which a lane has 16 bytes of the
// result's row and its neighbours the bytes beside them.  What is read from memory is requested before anything is stored.
template <typename T, typename TB, int TI, int TJ>
__device__ __forceinline__ void epilogue(f4 (&acc)[TI][TJ], const Plan& q, int act, const Place& at, int i0, int j0, float* mine)
{
    const dh_product& p = q.p;
    const int I = p.I, J = p.J, ob = at.batch, lane = threadIdx.x & 63;
    constexpr int V = Elem<T>::CH, W = TJ * 16, LANES = W / V, ROWS = 64 / LANES < 16 ? 64 / LANES : 16, PASSES = 16 / ROWS;
    constexpr int MASK = W / 4 - 1 < 15 ? W / 4 - 1 : 15;
    const int r = lane / LANES, jl = lane % LANES * V, j = j0 + jl;
    const bool live = j < J && r < ROWS, whole = j + V <= J;
    const bool joined = q.split > 1;                // partial sums: nothing but them, in fp32
    const T* bias = joined ? nullptr : (const T*)p.bias;
    const T* rp = joined ? nullptr : (const T*)p.residual;
    T* zp = joined ? nullptr : (T*)p.z;
    u4 res[TI][PASSES];
    float bi[TI][PASSES], bj[V];
    if (rp) {
        rp += (int64_t)ob * p.res_batch + j;
#pragma unroll
        for (int a = 0; a < TI; ++a)
#pragma unroll
            for (int n = 0; n < PASSES; ++n) {
                const int i = i0 + 16 * a + ROWS * n + r;
                res[a][n] = u4{0, 0, 0, 0};
                if (i < I && live) {
                    const T* from = rp + (int64_t)i * p.ldr;
                    if (whole) {
                        __builtin_memcpy(&res[a][n], from, 16);
                    } else {
                        T t[V];
                        __builtin_memset(t, 0, 16);
#pragma unroll
                        for (int e = 0; e < V - 1; ++e)
                            if (j + e < J) t[e] = from[e];
                        __builtin_memcpy(&res[a][n], t, 16);
                    }
                }
            }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) bj[e] = 0.f;
    if (bias && !p.bias_on_i) {
#pragma unroll
        for (int e = 0; e < V; ++e) bj[e] = Elem<T>::up(bias[j + e < J ? j + e : J - 1]);
    }
#pragma unroll
    for (int a = 0; a < TI; ++a)
#pragma unroll
        for (int n = 0; n < PASSES; ++n) {
            const int i = i0 + 16 * a + ROWS * n + r;
            bi[a][n] = bias && p.bias_on_i ? Elem<T>::up(bias[i < I ? i : I - 1]) : 0.f;
        }
#pragma unroll
    for (int a = 0; a < TI; ++a) {
        asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");        // the rows before have been read
#pragma unroll
        for (int b = 0; b < TJ; ++b) {
            const int m = lane & 15, c = TB::index(b, 4 * (lane >> 4)) / 4;
            *reinterpret_cast<f4*>(mine + m * W + (c ^ (m & MASK)) * 4) = acc[a][b];
        }
        asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");        // the wave's lanes read what its other lanes wrote
#pragma unroll
        for (int n = 0; n < PASSES; ++n) {
            const int row = ROWS * n + r, i = i0 + 16 * a + row;
            if (!live || i >= I) continue;
            float v[V];
#pragma unroll
            for (int h = 0; h < V / 4; ++h)
                *reinterpret_cast<f4*>(v + 4 * h) = *reinterpret_cast<const f4*>(mine + row * W + ((jl / 4 + h) ^ (row & MASK)) * 4);
            if (joined) {
                float* o = q.partial + (((int64_t)at.s * q.out_batches + ob) * I + i) * J + j;
                if (whole) __builtin_memcpy(o, v, 4 * V);
                else
#pragma unroll
                    for (int e = 0; e < V - 1; ++e)
                        if (j + e < J) o[e] = v[e];
                continue;
            }
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] += bi[a][n] + bj[e];          // (one of the two is zero)
            auto store = [&](T* o) {
                o += (int64_t)ob * p.o_batch + (int64_t)i * p.ldo + j;
                alignas(16) T t[V];
#pragma unroll
                for (int e = 0; e < V; ++e) t[e] = Elem<T>::down(v[e]);
                if (whole && q.stream) {
                    u4 w;
                    __builtin_memcpy(&w, t, 16);
                    __builtin_nontemporal_store(w, reinterpret_cast<u4*>(o));
                } else if (whole) {
                    __builtin_memcpy(o, t, 16);
                } else {
#pragma unroll
                    for (int e = 0; e < V - 1; ++e)
                        if (j + e < J) o[e] = t[e];
                }
            };
            if (zp) store(zp);
            with_act(act, [&](auto which) {
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] = Act<decltype(which)::value, sizeof(T) == 2>::value(v[e]);
            });
            if (rp) {
                T t[V];
                __builtin_memcpy(t, &res[a][n], 16);
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] += Elem<T>::up(t[e]);
            }
            store((T*)p.out);
        }
    }
}

// Aligned operands: a ring of STAGES buffers in LDS, the copies of STAGES - 1 steps on their way while one is multiplied (copied by
// the memory system itself, so that a step costs no registers and one barrier).
// Large reductions are bound by the matrix pipes: 8192^3 bf16 1357 TFLOP/s; with 1024 to reduce the prologue and the epilogue of
// a tile show, 8192 x 1024 -> 4096 bf16 71 us = 968 TFLOP/s, with gelu 81 (848).  Maps with few channels are bound by bytes: 128 ->
// 128 channels, silu and residual of 64 x 80 x 80 cells (315 MB) 75 us = 4.2 TB/s, where a plain copy of that card reaches 4.9.
template <typename T, int BI, int BJ, int BR, int WI, int WJ, int STAGES, int WAVES, bool ARC, bool BRC>
__global__ void __launch_bounds__(WI * WJ * 64, WAVES) k_product(const Launch L)
{
    constexpr int THREADS = WI * WJ * 64;
    constexpr int TI = BI / WI / 16, TJ = BJ / WJ / 16;
    typedef Stream<T, BI, BR, ARC, false, THREADS> SA;
    typedef Stream<T, BJ, BR, BRC, sizeof(T) == 2, THREADS> SB;
    typedef typename SA::TL TA;
    typedef typename SB::TL TB;
    static_assert(sizeof(T) == 4 || TJ % 2 == 0, "fragments of B go in pairs");
    __shared__ __align__(16) T lds[STAGES][(BI + BJ) * BR];

    Place at;
    if (!place(L, BI, BJ, &at)) return;
    const Plan& q = L.plan[at.w];
    const dh_product& p = q.p;
    const int k_begin = at.s * q.per, k_end = k_begin + q.per < q.steps ? k_begin + q.per : q.steps;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = (wave / WJ) * (BI / WI), wj = (wave % WJ) * (BJ / WJ);
    f4 acc[TI][TJ];
#pragma unroll
    for (int a = 0; a < TI; ++a)
#pragma unroll
        for (int b = 0; b < TJ; ++b) acc[a][b] = f4{0.f, 0.f, 0.f, 0.f};
    f4 rows[TI];
#pragma unroll
    for (int a = 0; a < TI; ++a) rows[a] = f4{0.f, 0.f, 0.f, 0.f};
    const bool sums = p.a_sum && at.j0 + wj == 0;

    SA sa;
    SB sb;
    int left = 0;                                    // reduction values of the current batch that are not requested yet
    int batch = at.batch, asked = k_begin;
    auto enter = [&](int r0) {
        sa.begin((const T*)p.a + (int64_t)batch * p.a_batch, p.lda, at.i0, p.I, r0);
        sb.begin((const T*)p.b + (int64_t)batch * p.b_batch, p.ldb, at.j0, p.J, r0);
        left = p.R - r0;
    };
    if (k_begin < k_end) {
        int r = k_begin;
        if (p.reduce_batch) {
            batch = k_begin / q.batch_steps;
            r -= batch * q.batch_steps;
        }
        enter(r * BR);
    }
    auto ask = [&]() {
        if (left <= 0) {                             // only a reduced batch has a next one
            ++batch;
            enter(0);
        }
        T* to = lds[(asked - k_begin) % STAGES] + wave * 64 * Elem<T>::CH;
        sa.copy(to, left);
        sb.copy(to + BI * BR, left);
        left -= BR;
        ++asked;
    };
#pragma unroll
    for (int k = 0; k < STAGES - 1; ++k)
        if (asked < k_end) ask();
    for (int k = k_begin; k < k_end; ++k) {
        if (asked - k == STAGES - 1) wait_and_meet<(STAGES - 2) * (SA::N + SB::N)>();
        else wait_and_meet<0>();
        if (asked < k_end) ask();
        const T* from = lds[(k - k_begin) % STAGES];
        multiply<T, TA, TB, BR, TI, TJ>(acc, rows, sums, from, from + BI * BR, wi, wj, lane);
    }
    static_assert(WI * WJ * TJ * 1024 <= (int)sizeof(lds), "room for the epilogue");
    __syncthreads();
    if (sums) row_sums<T, TI>(rows, q, at, at.i0 + wi);
    epilogue<T, TB, TI, TJ>(acc, q, L.act, at, at.i0 + wi, at.j0 + wj, (float*)lds + wave * TJ * 256);
}

// The reduction of one tile for operands of any alignment: one buffer in LDS behind DEPTH steps on their way in registers.
// `put` brings a step's registers to LDS, `take` multiplies what is there.  `groups` of threads share the steps of the tile (each
// a run of its own, with its own buffer); all of them pass the same barriers.
template <typename FA, typename FB, int BR, int DEPTH, typename Put, typename Take>
__device__ __forceinline__ void pass_over(const Plan& q, const Place& at, int group, int groups, Put&& put, Take&& take)
{
    const dh_product& p = q.p;
    typedef typename FA::type T;
    const int first = at.s * q.per, behind = first + q.per < q.steps ? first + q.per : q.steps;
    const int rounds = (behind - first + groups - 1) / groups;
    const int k_begin = first + group * rounds, k_end = k_begin + rounds < behind ? k_begin + rounds : behind;
    FA feed_a;
    FB feed_b;
    u4 ra[DEPTH][FA::N], rb[DEPTH][FB::N];
    int left = 0, batch = at.batch;
    auto enter = [&](int r0) {
        feed_a.begin((const T*)p.a + (int64_t)batch * p.a_batch, p.lda, at.i0, p.I, r0, p.R);
        feed_b.begin((const T*)p.b + (int64_t)batch * p.b_batch, p.ldb, at.j0, p.J, r0, p.R);
        left = p.R - r0;
    };
    if (k_begin < k_end) {
        int r = k_begin;
        if (p.reduce_batch) {
            batch = k_begin / q.batch_steps;
            r -= batch * q.batch_steps;
        }
        enter(r * BR);
    }
    auto fetch = [&](int d) {
        if (left <= 0) {
            ++batch;
            enter(0);
        }
        feed_a.fetch(ra[d], left);
        feed_b.fetch(rb[d], left);
        left -= BR;
    };
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
        if (k_begin + d < k_end) fetch(d);
    for (int k = k_begin; k < k_begin + rounds; k += DEPTH) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            if (k + d >= k_begin + rounds) break;
            __syncthreads();
            if (k + d < k_end) put(ra[d], rb[d]);
            __syncthreads();
            if (k + d + DEPTH < k_end) fetch(d);
            if (k + d < k_end) take();
        }
    }
}

template <int TI, int TJ> __device__ __forceinline__ void clear(f4 (&acc)[TI][TJ], f4 (&rows)[TI])
{
#pragma unroll
    for (int a = 0; a < TI; ++a) {
        rows[a] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int b = 0; b < TJ; ++b) acc[a][b] = f4{0.f, 0.f, 0.f, 0.f};
    }
}

// The groups' sums into the first group's registers, in the groups' order; `room`: (groups - 1) x THREADS x TI x (TJ + 1) f4 of LDS.
template <int TI, int TJ>
__device__ __forceinline__ void join_groups(f4 (&acc)[TI][TJ], f4 (&rows)[TI], int group, int groups, int threads, f4* room)
{
    const int tid = threadIdx.x & (threads - 1);
    __syncthreads();
    if (group) {
        f4* to = room + (group - 1) * threads * TI * (TJ + 1) + tid;
#pragma unroll
        for (int a = 0; a < TI; ++a) {
#pragma unroll
            for (int b = 0; b < TJ; ++b) to[(a * (TJ + 1) + b) * threads] = acc[a][b];
            to[(a * (TJ + 1) + TJ) * threads] = rows[a];
        }
    }
    __syncthreads();
    for (int g = 1; g < groups && !group; ++g) {
        const f4* from = room + (g - 1) * threads * TI * (TJ + 1) + tid;
#pragma unroll
        for (int a = 0; a < TI; ++a) {
#pragma unroll
            for (int b = 0; b < TJ; ++b) acc[a][b] += from[(a * (TJ + 1) + b) * threads];
            rows[a] += from[(a * (TJ + 1) + TJ) * threads];
        }
    }
    __syncthreads();
}

// Operands that the copies above cannot take (rows of a number of bytes that is no multiple of 16, unaligned pointers) and fp32 with
// less than 64 to reduce.  Bound by the instructions that bring a step to LDS: each 16 bytes pass through registers, with a shift
// where their row is not aligned.  8191 x 1023 -> 4095 bf16 134 us = 512 TFLOP/s, half of what the aligned neighbour reaches; 1023 x 777
// -> 1001 bf16 11.9 us, of which a 64 x 64 tile's 13 steps, one after another, are the most.
// GROUPS > 1: tiles that fill the chip only once are worked on by that many groups of waves, which share the reduction.
template <typename T, int BI, int BJ, int BR, int WI, int WJ, int DEPTH, int GROUPS, bool ARC, bool BRC>
__global__ void __launch_bounds__(WI * WJ * 64 * GROUPS) k_product_any(const Launch L)
{
    constexpr int THREADS = WI * WJ * 64;
    constexpr int TI = BI / WI / 16, TJ = BJ / WJ / 16;
    typedef Feed<T, BI, BR, ARC, false, THREADS> FA;
    typedef Feed<T, BJ, BR, BRC, sizeof(T) == 2, THREADS> FB;
    typedef typename FA::TL TA;
    typedef typename FB::TL TB;
    __shared__ __align__(16) T lds[GROUPS][(BI + BJ) * BR];
    const int group = GROUPS > 1 ? (int)threadIdx.x / THREADS : 0;
    T *lds_a = lds[group], *lds_b = lds_a + BI * BR;

    Place at;
    if (!place(L, BI, BJ, &at)) return;
    const Plan& q = L.plan[at.w];
    const int lane = threadIdx.x & 63, wave = (threadIdx.x & (THREADS - 1)) >> 6;
    const int wi = (wave / WJ) * (BI / WI), wj = (wave % WJ) * (BJ / WJ);
    f4 acc[TI][TJ], rows[TI];
    clear(acc, rows);
    const bool sums = q.p.a_sum && at.j0 + wj == 0;
    pass_over<FA, FB, BR, DEPTH>(
        q, at, group, GROUPS, [&](const u4* ra, const u4* rb) { FA::stage(lds_a, ra); FB::stage(lds_b, rb); },
        [&]() { multiply<T, TA, TB, BR, TI, TJ>(acc, rows, sums, lds_a, lds_b, wi, wj, lane); });
    static_assert(WI * WJ * TJ * 1024 <= (int)sizeof(lds), "room for the epilogue");
    if constexpr (GROUPS > 1) {
        static_assert((GROUPS - 1) * THREADS * TI * (TJ + 1) * 16 <= (int)sizeof(lds), "room for the join");
        join_groups(acc, rows, group, GROUPS, THREADS, (f4*)lds);
        if (group) return;
    } else {
        __syncthreads();
    }
    if (sums) row_sums<T, TI>(rows, q, at, at.i0 + wi);
    epilogue<T, TB, TI, TJ>(acc, q, L.act, at, at.i0 + wi, at.j0 + wj, (float*)lds + wave * TJ * 256);
}

// fp32 on the bf16 matrix instructions, whose rate is 16 times that of the fp32 ones: every value is split into three bf16 parts
// (x = hi + mid + lo to 2^-25 of x: each part holds the next 8 bits, rounded), and of the nine products of parts the six are
// formed that reach 2^-24 of the whole (hi hi, hi mid, mid hi, mid mid, hi lo, lo hi; the three left out are below 2^-23 together).
// A product of parts is exact in fp32 and sums are fp32, so this rounds where the fp32 instructions round.  What it cannot do is
// found out and done again with those: a part of an infinity or NaN, or of a value that rounds to an infinity in bf16, leaves a
// sum that is not finite; a part of a value below 2^-100 may underflow, which is looked for when the values are split.  Such a value
// is off by 2^-124 at most, its product by that times the other operand's largest: sums that reach 2^25 times what R of
// those add up to need nothing; the largest are found by another look at the operands, which only tiles that hold such a value take.
// (Underflowing gradients here and there in 8192 x 1024 -> 4096: 477 us against 374 without any, and 848 when every tile that holds one
// is done again.  Keeping the largest beside the split costs every tile 1.6 % and these 380.  Looking for small values at the first parts, which
// misses those below 2^-134, would be 0.7 % faster.)
// Six products at 1/16 of the cost each: at best 2.7 times the fp32 rate; the split costs 7 vector instructions per value and
// tile, which other workgroups' products hide.
struct Split {
    u2 hi, mid, lo;         // four values' parts
};
__device__ __forceinline__ Split split(u4 v, uint32_t* smallest)
{
    Split s;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const f2 x = {__uint_as_float(v[2 * h]), __uint_as_float(v[2 * h + 1])};
        const uint32_t hi = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, b2));
        const f2 r = {x[0] - __uint_as_float(hi << 16), x[1] - __uint_as_float(hi & 0xFFFF0000u)};
        const uint32_t mid = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, b2));
        const f2 t = {r[0] - __uint_as_float(mid << 16), r[1] - __uint_as_float(mid & 0xFFFF0000u)};
        s.hi[h] = hi;
        s.mid[h] = mid;
        s.lo[h] = __builtin_bit_cast(uint32_t, __builtin_convertvector(t, b2));
        // the smallest magnitude but zero, from the value itself (below 2^-134 its first part is zero too): twice its bits, which
        // leaves the sign behind, less one; 0 - 1 is the largest number there is
        *smallest = min(*smallest, min((v[2 * h] << 1) - 1, (v[2 * h + 1] << 1) - 1));
    }
    return s;
}

// The largest magnitude in a wave's values (a NaN is passed over: its sums are done again anyway).
template <int N> __device__ __forceinline__ void most_of(const u4* v, float* most)
{
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) *most = fmaxf(*most, fabsf(__uint_as_float(v[k][e])));
}
__device__ __forceinline__ float wave_most(float v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}

// fp32 products, six bf16 ones each (above).  Long reductions are bound by the vector instructions that split beside the matrix
// instructions that multiply: 8192 x 1024 -> 4096 366 us = 188 TFLOP/s, 8192^3 198, where the card's fp32 matrix instructions end at
// 157.  The head's levels at batch 64 (548 MB of 915 written) take 404 us: 266 of memory and 283 of products, which overlap between
// the two workgroups of a CU only in part.  Few tiles (1023 x 777 -> 1001, 23 us) wait for their steps one by one.
template <int BI, int BJ, int WI, int WJ, int DEPTH, int WAVES, int GROUPS, bool ARC, bool BRC>
__global__ void __launch_bounds__(WI * WJ * 64 * GROUPS, WAVES) k_product_split(const Launch L)
{
    constexpr int THREADS = WI * WJ * 64, BR = 32;
    constexpr int TI = BI / WI / 16, TJ = BJ / WJ / 16;
    typedef Feed<float, BI, BR, ARC, false, THREADS> FA;
    typedef Feed<float, BJ, BR, BRC, false, THREADS> FB;
    typedef Tile<__bf16, BI, BR, ARC, false> TA;
    typedef Tile<__bf16, BJ, BR, BRC, false> TB;
    __shared__ __align__(16) __bf16 lds[GROUPS][3 * (BI + BJ) * BR];       // hi, mid, lo of A, then of B
    const int group = GROUPS > 1 ? (int)threadIdx.x / THREADS : 0;
    __bf16 *la = lds[group], *lb = la + 3 * BI * BR;

    Place at;
    if (!place(L, BI, BJ, &at)) return;
    const Plan& q = L.plan[at.w];
    const int tid = threadIdx.x & (THREADS - 1), lane = threadIdx.x & 63, wave = tid >> 6;
    const int wi = (wave / WJ) * (BI / WI), wj = (wave % WJ) * (BJ / WJ);
    f4 acc[TI][TJ], rows[TI];
    clear(acc, rows);
    const bool sums = q.p.a_sum && at.j0 + wj == 0;
    uint32_t smallest = 0xFFFFFFFFu;
    auto put_one = [&](auto tile, __bf16* to, int plane, int k, u4 v) {
        typedef decltype(tile) TL;
        constexpr int ROW = TL::ROW_CHUNKS * 2;                     // 4-value pieces in a row
        const int row = k / ROW, c = k % ROW;
        __bf16* o = to + (row * TL::ROW_CHUNKS + ((c >> 1) ^ TL::key(row))) * 8 + (c & 1) * 4;
        const Split s = split(v, &smallest);
        *reinterpret_cast<u2*>(o) = s.hi;
        *reinterpret_cast<u2*>(o + plane) = s.mid;
        *reinterpret_cast<u2*>(o + 2 * plane) = s.lo;
    };
    pass_over<FA, FB, BR, DEPTH>(
        q, at, group, GROUPS,
        [&](const u4* ra, const u4* rb) {
#pragma unroll
            for (int k = 0; k < FA::N; ++k) put_one(TA(), la, BI * BR, k * THREADS + tid, ra[k]);
#pragma unroll
            for (int k = 0; k < FB::N; ++k) put_one(TB(), lb, BJ * BR, k * THREADS + tid, rb[k]);
        },
        [&]() {
            s8 fb[TJ][3], ones;
#pragma unroll
            for (int e = 0; e < 8; ++e) ones[e] = 0x3F80;
#pragma unroll
            for (int b = 0; b < TJ; ++b)
#pragma unroll
                for (int h = 0; h < 3; ++h) fb[b][h] = TB::frag16(lb + h * BJ * BR, wj, b, 0, lane);
            // the small products first; GROUP rows of fragments at a time keep products into one accumulator four apart
            constexpr int GROUP = TJ >= 4 ? 1 : 4 / TJ;
#pragma unroll
            for (int a0 = 0; a0 < TI; a0 += GROUP) {
                s8 fa[GROUP][3];
#pragma unroll
                for (int a = 0; a < GROUP; ++a)
#pragma unroll
                    for (int h = 0; h < 3; ++h) fa[a][h] = TA::frag16(la + h * BI * BR, wi, a0 + a, 0, lane);
                constexpr int pa[6] = {0, 2, 1, 0, 1, 0}, pb[6] = {2, 0, 1, 1, 0, 0};
#pragma unroll
                for (int h = 0; h < 6; ++h)
#pragma unroll
                    for (int a = 0; a < GROUP; ++a)
#pragma unroll
                        for (int b = 0; b < TJ; ++b) acc[a0 + a][b] = mma16<__bf16>(fb[b][pb[h]], fa[a][pa[h]], acc[a0 + a][b]);
                if (sums) {
#pragma unroll
                    for (int a = 0; a < GROUP; ++a)
#pragma unroll
                        for (int h = 2; h >= 0; --h) rows[a0 + a] = mma16<__bf16>(ones, fa[a][h], rows[a0 + a]);
                }
            }
        });
    const bool tiny = smallest < (0x0D800000u << 1) - 1;            // the bits of 2^-100
    bool again = false;
#pragma unroll
    for (int a = 0; a < TI; ++a) {
#pragma unroll
        for (int b = 0; b < TJ; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) again |= !(fabsf(acc[a][b][e]) <= 3.402823466e38f);
        again |= !(fabsf(rows[a][0]) <= 3.402823466e38f);
    }
    again = __syncthreads_or(again || tiny) && [&]() {              // (the same in every thread, from here on)
        if (__syncthreads_or(again)) return true;
        float largest_a = 0.f, largest_b = 0.f;
        pass_over<FA, FB, BR, 1>(
            q, at, group, GROUPS, [&](const u4* ra, const u4* rb) { most_of<FA::N>(ra, &largest_a); most_of<FB::N>(rb, &largest_b); }, []() {});
        float(*most)[2] = (float(*)[2])lds;
        const float a_wave = wave_most(largest_a), b_wave = wave_most(largest_b);
        if (lane == 0) {
            most[threadIdx.x >> 6][0] = a_wave;
            most[threadIdx.x >> 6][1] = b_wave;
        }
        __syncthreads();
        float most_a = 0.f, most_b = 0.f;
        for (int w = 0; w < THREADS * GROUPS / 64; ++w) {
            most_a = fmaxf(most_a, most[w][0]);
            most_b = fmaxf(most_b, most[w][1]);
        }
        const float off = (float)q.per * BR * 0x1p-99f, least = off * (most_a + most_b);
        bool small = false;
#pragma unroll
        for (int a = 0; a < TI; ++a) {
            const bool row = at.i0 + wi + 16 * a + (lane & 15) < q.p.I;
#pragma unroll
            for (int b = 0; b < TJ; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    small |= row && at.j0 + wj + TB::index(b, 4 * (lane >> 4) + e) < q.p.J && !(fabsf(acc[a][b][e]) >= least);
            small |= sums && row && !(fabsf(rows[a][0]) >= off);
        }
        return __syncthreads_or(small) != 0;
    }();
    if (again) {
        typedef typename FA::TL NA;
        typedef typename FB::TL NB;
        float *na = (float*)la, *nb = na + BI * BR;
        clear(acc, rows);
        pass_over<FA, FB, BR, 1>(
            q, at, group, GROUPS, [&](const u4* ra, const u4* rb) { FA::stage(na, ra); FB::stage(nb, rb); },
            [&]() { multiply<float, NA, NB, BR, TI, TJ>(acc, rows, sums, na, nb, wi, wj, lane); });
        __syncthreads();
    }
    if constexpr (GROUPS > 1) {
        static_assert((GROUPS - 1) * THREADS * TI * (TJ + 1) * 16 <= (int)sizeof(lds), "room for the join");
        join_groups(acc, rows, group, GROUPS, THREADS, (f4*)lds);
        if (group) return;
    }
    static_assert(WI * WJ * TJ * 1024 <= (int)sizeof(lds), "room for the epilogue");
    if (sums) row_sums<float, TI>(rows, q, at, at.i0 + wi);
    epilogue<float, TB, TI, TJ>(acc, q, L.act, at, at.i0 + wi, at.j0 + wj, (float*)lds + wave * TJ * 256);
}

// One value of C through the epilogue.
template <typename T> __device__ __forceinline__ void finish_one(const dh_product& p, int act, int b, int i, int j, float v)
{
    if (p.bias) v += Elem<T>::up(((const T*)p.bias)[p.bias_on_i ? i : j]);
    const int64_t o = (int64_t)b * p.o_batch + (int64_t)i * p.ldo + j;
    if (p.z) ((T*)p.z)[o] = Elem<T>::down(v);
    with_act(act, [&](auto a) { v = Act<decltype(a)::value, sizeof(T) == 2>::value(v); });
    if (p.residual) v += Elem<T>::up(((const T*)p.residual)[(int64_t)b * p.res_batch + (int64_t)i * p.ldr + j]);
    ((T*)p.out)[o] = Elem<T>::down(v);
}

// Few rows of A (tokens) against many of B (a weight): bound by reading B once.  A workgroup of 8 waves takes 16 rows of B; its
// waves take the reduction in turns of 128 bytes, fragments come from memory straight into registers (no row is used twice, so
// LDS would only add a trip), and the waves' sums are added in order at the end.  Lane (m, g) reads 32 consecutive bytes of row
// m, for two products of which each pairs the same reduction values of A and B; which values those are does not matter.
// Short products of more rows take it too, 64 rows to a workgroup.
// One token, 4096 -> 16384 bf16: 24 us = 5.5 TB/s of weight; 4096 -> 4096 7.1 us = 4.7 TB/s (and 16 tokens 9.4).
constexpr int THIN_ROWS = 64;           // of A that a workgroup takes (16 MI, where there are no more)
template <typename T, int MI>
__global__ void __launch_bounds__(512) k_product_thin(const Launch L)
{
    constexpr int CH = Elem<T>::CH, TURN = 8 * CH, WAVES = 8, AHEAD = 4 / MI;
    __shared__ float sums[WAVES][MI * 256];
    const Plan& q = L.plan[0];
    const dh_product& p = q.p;
    const int tile = (int)blockIdx.x % q.tiles_j, rest = (int)blockIdx.x / q.tiles_j, ob = rest / q.tiles_i, i0 = rest % q.tiles_i * THIN_ROWS;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, g = lane >> 4, R = p.R, j0 = tile * 16;
    const T* b = (const T*)p.b + (int64_t)ob * p.b_batch + (int64_t)(j0 + m < p.J ? j0 + m : p.J - 1) * p.ldb;
    const T* a[MI];
#pragma unroll
    for (int n = 0; n < MI; ++n)
        a[n] = (const T*)p.a + (int64_t)ob * p.a_batch + (int64_t)(i0 + 16 * n + m < p.I ? i0 + 16 * n + m : p.I - 1) * p.lda;
    f4 acc[MI];
#pragma unroll
    for (int n = 0; n < MI; ++n) acc[n] = f4{0.f, 0.f, 0.f, 0.f};

    auto multiply = [&](const u4 (&vb)[2], const u4 (&va)[MI][2]) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int n = 0; n < MI; ++n) {
                if constexpr (sizeof(T) == 4) {
                    const f4 fb = __builtin_bit_cast(f4, vb[h]), fa = __builtin_bit_cast(f4, va[n][h]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[e], fa[e], acc[n], 0, 0, 0);
                } else {
                    acc[n] = mma16<T>(__builtin_bit_cast(s8, vb[h]), __builtin_bit_cast(s8, va[n][h]), acc[n]);
                }
            }
    };
    // the 2 CH values at k of a row; with an end: zeros from there on
    auto whole = [&](const T* row, int k, u4 (&v)[2]) {
        __builtin_memcpy(&v[0], row + k, 16);
        __builtin_memcpy(&v[1], row + k + CH, 16);
    };
    auto some = [&](const T* row, int k, int end, u4 (&v)[2]) {
        T e[2 * CH];
#pragma unroll
        for (int x = 0; x < 2 * CH; ++x) e[x] = k + x < end ? row[k + x] : T(0);
        __builtin_memcpy(&v[0], e, 16);
        __builtin_memcpy(&v[1], e + CH, 16);
    };
    const int turns = R / TURN;
    int t = wave;
    for (; t + (AHEAD - 1) * WAVES < turns; t += AHEAD * WAVES) {
        u4 vb[AHEAD][2], va[AHEAD][MI][2];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int k = (t + u * WAVES) * TURN + g * 2 * CH;
            whole(b, k, vb[u]);
#pragma unroll
            for (int n = 0; n < MI; ++n) whole(a[n], k, va[u][n]);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) multiply(vb[u], va[u]);
    }
    for (; t < turns; t += WAVES) {
        u4 vb[2], va[MI][2];
        const int k = t * TURN + g * 2 * CH;
        whole(b, k, vb);
#pragma unroll
        for (int n = 0; n < MI; ++n) whole(a[n], k, va[n]);
        multiply(vb, va);
    }
    if (t == turns && turns * TURN < R) {        // the wave whose turn it is takes what remains
        u4 vb[2], va[MI][2];
        const int k = t * TURN + g * 2 * CH;
        some(b, k, R, vb);
#pragma unroll
        for (int n = 0; n < MI; ++n) some(a[n], k, R, va[n]);
        multiply(vb, va);
    }
#pragma unroll
    for (int n = 0; n < MI; ++n) *reinterpret_cast<f4*>(&sums[wave][n * 256 + m * 16 + 4 * g]) = acc[n];
    __syncthreads();
    for (int k = threadIdx.x; k < MI * 256; k += 512) {
        const int i = i0 + k / 16, j = j0 + k % 16;
        if (i >= p.I || j >= p.J) return;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) v += sums[w][k];
        finish_one<T>(p, L.act, ob, i, j, v);
    }
}

// Sums the partial products of the workgroups along the reduction, in a fixed order, and finishes them.  A thread adds four
// values' parts, eight requested at a time; with many parts, eight threads share them (every eighth part each) and their sums are
// added in turn.  All products of a launch that were split join in one launch.  Bound by the trip to memory: 17 MB of parts, the
// head's weight gradients at batch 64, 12 us beside 101 for their products.
struct Joins {
    int w[DH_MAX_PRODUCTS], first[DH_MAX_PRODUCTS + 1], n;
    int share[DH_MAX_PRODUCTS];             // 1 or 8 threads per value
};
template <typename T>
__global__ void __launch_bounds__(256) k_product_join(const Launch L, const Joins js)
{
    __shared__ f4 shared[256];
    int k = 0;
    while (k + 1 < js.n && (int)blockIdx.x >= js.first[k + 1]) ++k;
    const Plan& q = L.plan[js.w[k]];
    const dh_product& p = q.p;
    const int share = js.share[k], wide = 256 / share, part = (int)threadIdx.x / wide;
    const int64_t n = (int64_t)q.out_batches * p.I * p.J, quads = (n + 3) / 4;
    const int64_t quad = (int64_t)((int)blockIdx.x - js.first[k]) * wide + threadIdx.x % wide, at = quad * 4;
    const bool products = quad < quads;
    f4 v = {0.f, 0.f, 0.f, 0.f};
    if (products) {
        const float* from = q.partial + at;
        if (at + 4 <= n) {
            int s = part;
            for (; s + 7 * share < q.split; s += 8 * share) {
                f4 t[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) __builtin_memcpy(&t[u], from + (int64_t)(s + u * share) * n, 16);
#pragma unroll
                for (int u = 0; u < 8; ++u) v += t[u];
            }
            for (; s < q.split; s += share) {
                f4 t;
                __builtin_memcpy(&t, from + (int64_t)s * n, 16);
                v += t;
            }
        } else {
            for (int s = part; s < q.split; s += share)
#pragma unroll
                for (int e = 0; e < 3; ++e)
                    if (at + e < n) v[e] += from[(int64_t)s * n + e];
        }
    } else if (p.a_sum && quad - quads < p.I) {       // behind the products: the row sums, one each
        for (int s = part; s < q.split; s += share) v[0] += q.partial_sum[(int64_t)s * p.I + quad - quads];
    }
    if (share > 1) {                        // uniform in the workgroup
        shared[threadIdx.x] = v;
        __syncthreads();
        if (part) return;
        for (int u = 1; u < share; ++u) v += shared[u * wide + threadIdx.x];
    }
    if (!products) {
        if (p.a_sum && quad - quads < p.I) ((T*)p.a_sum)[quad - quads] = Elem<T>::down(v[0]);
        return;
    }
    int64_t rest = at / p.J;
    int j = (int)(at - rest * p.J), b = (int)(rest / p.I), i = (int)(rest - (int64_t)b * p.I);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (at + e >= n) break;
        finish_one<T>(p, L.act, b, i, j, v[e]);
        if (++j == p.J) {
            j = 0;
            if (++i == p.I) { i = 0; ++b; }
        }
    }
}

constexpr int CUS = 256;
constexpr int SPLIT = -1;              // stages of a shape whose fp32 values are split
// br: bytes of a reduction step's row; bi = 0: the thin kernel; groups: of waves that share a tile's reduction
struct Shape { int bi, bj, br, stages, groups = 1; };

// Tiles (i, j), bytes of a reduction step, waves along i and j, stages of the ring, waves per SIMD
#define DH_SHAPES(X) X(128, 128, 128, 2, 2, 2, 2) X(128, 128, 64, 2, 2, 3, 3) X(64, 64, 128, 2, 2, 2, 4) X(64, 64, 128, 2, 2, 4, 2)
#define DH_SHAPES_16(X) X(256, 256, 128, 2, 4, 2, 2)

template <typename T, bool ARC, bool BRC>
void launch_tiles(const Launch& L, bool aligned, const Shape& t, hipStream_t st)
{
    constexpr int BR = 128 / sizeof(T);
    const dim3 grid((unsigned)L.total);
    if (t.bi == 0) {
        if constexpr (ARC && BRC) {
            const dim3 all((unsigned)L.plan[0].count);
            if (L.plan[0].p.I <= 16) hipLaunchKernelGGL((k_product_thin<T, 1>), all, dim3(512), 0, st, L);
            else if (L.plan[0].p.I <= 32) hipLaunchKernelGGL((k_product_thin<T, 2>), all, dim3(512), 0, st, L);
            else hipLaunchKernelGGL((k_product_thin<T, 4>), all, dim3(512), 0, st, L);
        }
        return;
    }
    if (aligned && t.stages != SPLIT) {
#define DH_CASE(BI, BJ, BYTES, WI, WJ, STAGES, WAVES) \
        if (t.bi == BI && t.bj == BJ && t.br == BYTES && t.stages == STAGES) { \
            hipLaunchKernelGGL((k_product<T, BI, BJ, BYTES / (int)sizeof(T), WI, WJ, STAGES, WAVES, ARC, BRC>), grid, dim3(WI * WJ * 64), 0, \
                               st, L); \
            return; \
        }
        DH_SHAPES(DH_CASE)
        if constexpr (sizeof(T) == 2) {
            DH_SHAPES_16(DH_CASE)
        }
#undef DH_CASE
        return;
    }
    if constexpr (sizeof(T) == 4) {
        if (t.stages == SPLIT) {
            if (t.bi == 128) hipLaunchKernelGGL((k_product_split<128, 128, 2, 2, 1, 2, 1, ARC, BRC>), grid, dim3(256), 0, st, L);
            else if (t.groups == 2) hipLaunchKernelGGL((k_product_split<64, 64, 2, 2, 2, 2, 2, ARC, BRC>), grid, dim3(512), 0, st, L);
            else hipLaunchKernelGGL((k_product_split<64, 64, 2, 2, 2, 3, 1, ARC, BRC>), grid, dim3(256), 0, st, L);
            return;
        }
    }
    if (t.bi == 128) hipLaunchKernelGGL((k_product_any<T, 128, 128, BR, 2, 2, 1, 1, ARC, BRC>), grid, dim3(256), 0, st, L);
    else if (t.groups == 2) hipLaunchKernelGGL((k_product_any<T, 64, 64, BR, 2, 2, 2, 2, ARC, BRC>), grid, dim3(512), 0, st, L);
    else hipLaunchKernelGGL((k_product_any<T, 64, 64, BR, 2, 2, 2, 1, ARC, BRC>), grid, dim3(256), 0, st, L);
}

template <typename T>
int launch(const Launch& L, bool arc, bool brc, bool aligned, const Shape& t, hipStream_t st)
{
    if (L.total > 0) {
        if (arc && brc) launch_tiles<T, true, true>(L, aligned, t, st);
        else if (arc) launch_tiles<T, true, false>(L, aligned, t, st);
        else launch_tiles<T, false, false>(L, aligned, t, st);
    }
    Joins js;
    js.n = 0;
    int64_t blocks = 0;
    for (int w = 0; w < L.n; ++w) {
        const Plan& q = L.plan[w];
        if (q.split <= 1) continue;
        const int64_t n = (int64_t)q.out_batches * q.p.I * q.p.J, threads = (n + 3) / 4 + (q.p.a_sum ? q.p.I : 0);
        const int share = q.split >= 32 ? 8 : 1;
        js.w[js.n] = w;
        js.share[js.n] = share;
        js.first[js.n++] = (int)blocks;
        blocks += (threads * share + 255) / 256;
    }
    js.first[js.n] = (int)blocks;
    if (blocks >= (1ll << 31)) return DH_ERR_ARG;
    if (js.n) hipLaunchKernelGGL((k_product_join<T>), dim3((unsigned)blocks), dim3(256), 0, st, L, js);
    return dh_launch_status();
}

// ---- dz = dy * act'(z) and the bias gradient ----
// dy is [outer][n][inner]; the bias gradient sums over outer and inner.  One pass over dy and z in 16-byte pieces (of any
// alignment): a wave takes rows of `inner` values of one n (maps), or the same 64 pieces of columns in every row (inner = 1).
// Sums go to the workspace, SPLIT of them at most per n, and are added in order by k_bias_join.
// Two roundings to 16 bits are choices: z is kept in the tensors' type between forward and backward (in fp32 it would be half of what a
// forward pass with an activation writes and the slope reads again), and dz is rounded to it because the matrix instructions that
// read it take 16 bits; the bias gradient sums it before that.  Gradients are then off by two half steps instead of one: 8192 x 1024 ->
// 1024 bf16 0.0024 from 64 bits, 0.0017 with both in fp32.
constexpr int BIAS_SPLIT = 256;

// v[k] = dy * act'(z), stored where dz is; the values count from `at` in one piece of V, `n` of them exist
template <typename T, int V>
__device__ __forceinline__ void slope_piece(const T* dy, const T* z, T* dz, int64_t at, int n, int act, float* v)
{
    T g[V], y[V];
    const bool whole = n >= V;
    if (whole) {
        __builtin_memcpy(g, dy + at, 16);
        if (z) __builtin_memcpy(y, z + at, 16);
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            g[k] = k < n ? dy[at + k] : T(0);
            y[k] = z && k < n ? z[at + k] : T(0);
        }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = Elem<T>::up(g[k]);
    if (!z) return;
    with_act(act, [&](auto a) {
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = act_back<decltype(a)::value, sizeof(T) == 2>(v[k], Elem<T>::up(y[k]));
    });
#pragma unroll
    for (int k = 0; k < V; ++k) g[k] = Elem<T>::down(v[k]);
    if (whole) {
        __builtin_memcpy(dz + at, g, 16);
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (k < n) {
                dz[at + k] = g[k];
            } else {
                v[k] = 0.f;         // (dy is 0 there, but the slope at 0 need not be finite times 0)
            }
    }
}

// U whole pieces `apart` from each other, all requested before the first is used: 16 values per thread, with twice that the registers
// allow fewer waves.  Maps: 64 x 128 x 80 x 80 bf16 55 us = 5.7 TB/s against 72 one by one, 64 x 256 x 40 x 40 30 against 38; fp32
// 127 = 4.9 TB/s against 133.  Rows gain nothing from it (8192 x 4096 bf16 36 us = 5.6 TB/s).
template <typename T, int V, int U>
__device__ __forceinline__ void slope_pieces(const T* dy, const T* z, T* dz, int64_t at, int apart, int act, float (&v)[U][V])
{
    T g[U][V], y[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) __builtin_memcpy(g[u], dy + at + u * apart, 16);
    if (z) {
#pragma unroll
        for (int u = 0; u < U; ++u) __builtin_memcpy(y[u], z + at + u * apart, 16);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < V; ++k) v[u][k] = Elem<T>::up(g[u][k]);
    if (!z) return;
    with_act(act, [&](auto a) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < V; ++k) v[u][k] = act_back<decltype(a)::value, sizeof(T) == 2>(v[u][k], Elem<T>::up(y[u][k]));
    });
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int k = 0; k < V; ++k) g[u][k] = Elem<T>::down(v[u][k]);
        __builtin_memcpy(dz + at + u * apart, g[u], 16);
    }
}

template <typename T>
__global__ void __launch_bounds__(256) k_slope_planes(const T* __restrict__ dy, const T* __restrict__ z, T* __restrict__ dz,
                                                      float* __restrict__ partial, int64_t outer, int64_t n, int64_t inner, int act, int split)
{
    constexpr int V = Elem<T>::CH;
    const int64_t c = blockIdx.x % n, s = blockIdx.x / n;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float sum = 0.f;
    for (int64_t o = s * 4 + wave; o < outer; o += 4 * split) {
        const int64_t row = (o * n + c) * inner;
        constexpr int U = 16 / V;
        int64_t k = lane * V;
        for (; k + ((U - 1) * 64 + 1) * V <= inner; k += U * 64 * V) {
            float v[U][V];
            slope_pieces<T, V, U>(dy, z, dz, row + k, 64 * V, act, v);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < V; ++e) sum += v[u][e];
        }
        for (; k < inner; k += 64 * V) {
            float v[V];
            slope_piece<T, V>(dy, z, dz, row + k, inner - k < V ? (int)(inner - k) : V, act, v);
#pragma unroll
            for (int e = 0; e < V; ++e) sum += v[e];
        }
    }
    if (!partial) return;
    __shared__ float sums[4];
    sum = dh_wave_sum(sum);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) partial[s * n + c] = sums[0] + sums[1] + sums[2] + sums[3];
}

template <typename T>
__global__ void __launch_bounds__(256) k_slope_rows(const T* __restrict__ dy, const T* __restrict__ z, T* __restrict__ dz,
                                                    float* __restrict__ partial, int64_t rows, int64_t n, int act, int split)
{
    constexpr int V = Elem<T>::CH;
    __shared__ float sums[4][64 * V];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t columns = (n + 64 * V - 1) / (64 * V);
    const int64_t c = blockIdx.x % columns * 64 * V + lane * V, s = blockIdx.x / columns;
    const int here = n - c < V ? (int)(n - c) : V;
    float sum[V];
#pragma unroll
    for (int e = 0; e < V; ++e) sum[e] = 0.f;
    if (c < n)
#pragma unroll 4
        for (int64_t r = s * 4 + wave; r < rows; r += 4 * split) {
            float v[V];
            slope_piece<T, V>(dy, z, dz, r * n + c, here, act, v);
#pragma unroll
            for (int e = 0; e < V; ++e) sum[e] += v[e];
        }
    if (!partial) return;
#pragma unroll
    for (int e = 0; e < V; ++e) sums[wave][lane * V + e] = sum[e];
    __syncthreads();
    for (int k = threadIdx.x; k < 64 * V; k += 256) {
        const int64_t at = blockIdx.x % columns * 64 * V + k;
        if (at < n) partial[s * n + at] = sums[0][k] + sums[1][k] + sums[2][k] + sums[3][k];
    }
}

// 32 sums per workgroup, eight threads for each
template <typename T>
__global__ void __launch_bounds__(256) k_bias_join(const float* __restrict__ partial, T* __restrict__ dbias, int64_t n, int split)
{
    __shared__ float shared[256];
    const int64_t c = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
    const int part = threadIdx.x >> 5;
    float sum = 0.f;
    if (c < n)
#pragma unroll 4
        for (int s = part; s < split; s += 8) sum += partial[s * n + c];
    shared[threadIdx.x] = sum;
    __syncthreads();
    if (part || c >= n) return;
    for (int u = 1; u < 8; ++u) sum += shared[u * 32 + threadIdx.x];
    dbias[c] = Elem<T>::down(sum);
}

template <typename T>
int launch_slope(const void* dy, const void* z, void* dz, void* dbias, int64_t outer, int64_t n, int64_t inner, int act,
                 float* ws, hipStream_t st)
{
    float* partial = dbias ? ws : nullptr;
    // about 2048 workgroups, each with four rows or more
    const int64_t columns = inner > 1 ? n : (n + 64 * Elem<T>::CH - 1) / (64 * Elem<T>::CH);
    int64_t split = (2048 + columns - 1) / columns;
    if (split > (outer + 3) / 4) split = (outer + 3) / 4;
    if (split > BIAS_SPLIT) split = BIAS_SPLIT;
    if (split < 1) split = 1;
    if (outer == 0 || inner == 0)               // nothing to read: dbias becomes the sum of no parts
        split = 0;
    else if (inner > 1)
        hipLaunchKernelGGL((k_slope_planes<T>), dim3((unsigned)(columns * split)), dim3(256), 0, st, (const T*)dy, (const T*)z, (T*)dz,
                           partial, outer, n, inner, act, (int)split);
    else
        hipLaunchKernelGGL((k_slope_rows<T>), dim3((unsigned)(columns * split)), dim3(256), 0, st, (const T*)dy, (const T*)z,
                           (T*)dz, partial, outer, n, act, (int)split);
    if (dbias)
        hipLaunchKernelGGL((k_bias_join<T>), dim3((unsigned)((n + 31) / 32)), dim3(256), 0, st, partial, (T*)dbias, n, (int)split);
    return dh_launch_status();
}


// One element type each in product_f32.hip, product_f16.hip and product_bf16.hip, which build side by side.
extern template int launch<float>(const Launch&, bool, bool, bool, const Shape&, hipStream_t);
extern template int launch<_Float16>(const Launch&, bool, bool, bool, const Shape&, hipStream_t);
extern template int launch<__bf16>(const Launch&, bool, bool, bool, const Shape&, hipStream_t);
extern template int launch_slope<float>(const void*, const void*, void*, void*, int64_t, int64_t, int64_t, int, float*, hipStream_t);
extern template int launch_slope<_Float16>(const void*, const void*, void*, void*, int64_t, int64_t, int64_t, int, float*, hipStream_t);
extern template int launch_slope<__bf16>(const void*, const void*, void*, void*, int64_t, int64_t, int64_t, int, float*, hipStream_t);

}  // namespace dhp
