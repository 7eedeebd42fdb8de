// The C entries of the matrix products: checks, how a launch is cut, and the dispatch by type (kernels in dh_product.h).
#include "dh_product.h"

using namespace dhp;

namespace {

// The tile of a launch, by what it measured (us, bf16):
//   256 x 256 (one workgroup of 8 waves per CU) where two of them per CU exist, they are at least 7/8 full and the reduction is
//     long enough to pay for filling them: 8192 x 1024 -> 4096 72 against 83, 512 -> 256 channels of 64 x 80 x 80 cells 181 against
//     210; but 128 -> 256 channels 95 against 76.
//   128 x 128 in steps of 128 bytes and 2 stages where the reduction is long: 8192 x 4096 -> 1024 66 against 78; in steps of 64
//     bytes and 3 stages (48 KB: three workgroups per CU) where it is short and loading, multiplying and storing have to
//     overlap between workgroups: the head's levels (128 to 512 channels) at batch 64 119 against 159.
//   64 x 64 where 128 x 128 would leave CUs without a tile, unless the reduction can be cut into 16 or more steps for two
//     workgroups per CU: the head's weight gradients at batch 64 (14 tiles, 44 steps each) 117 against 155, 1024 x 1024 over 8192 rows
//     (16 steps) 34 against 45; but 128 x 128 over 64 x 80 x 80 cells (12 steps) 56 against 40.  Their ring has 4 stages where there are two
//     of them per CU at most and a step waits for memory (256 x 4096 -> 4096 26 against 35, 1024 x 4096 -> 1024 26 against 35), 2
//     where more than two share a CU, whose LDS would hold no more of the deep ones (1024 x 1024 -> 2880, 720 tiles: 14 against 19).
Shape shape_of(const dh_product* ps, int n, int dtype, bool aligned)
{
    int64_t huge = 0, large = 0, small = 0, held = 0, tile_steps = 0;
    const int64_t br = dtype == DH_F32 ? 32 : 64;
    int longest = 0, shortest = 1 << 30;
    for (int w = 0; w < n; ++w) {
        const int64_t b = ps[w].reduce_batch ? 1 : ps[w].batch;
        huge += (int64_t)((ps[w].I + 255) / 256) * ((ps[w].J + 255) / 256) * b;
        const int64_t tiles = (int64_t)((ps[w].I + 127) / 128) * ((ps[w].J + 127) / 128) * b;
        large += tiles;
        small += (int64_t)((ps[w].I + 63) / 64) * ((ps[w].J + 63) / 64) * b;
        tile_steps += tiles * ((ps[w].R + br - 1) / br) * (ps[w].reduce_batch ? ps[w].batch : 1);
        held += (int64_t)ps[w].I * ps[w].J * b;
        if (ps[w].R > longest) longest = ps[w].R;
        if (ps[w].R < shortest) shortest = ps[w].R;
    }
    // thin: one product, both operands along the reduction.  At most 32 rows, and enough groups of 16 outputs for half the CUs, or rows
    // so short that a workgroup is done with all of them soon (us, bf16: 1 x 4096 -> 1024 6.7 against 9.6 on tiles, 32 x 1000 -> 777 4.8
    // against 10.3, 1 x 512 -> 512 2.9 against 6.2, fp32 3.6 against 13.9; but 32 x 4096 -> 1024 13 against 10, 1 x 16384 -> 16 19 against 10).
    // More rows, in groups of 64, where the reduction is short and the CUs hold all groups at once (64 x 512 -> 512 bf16 5.2 against 6.6,
    // fp32 7.6 against 15.0; 256 x 1024 -> 1024 7.8 against 9.4, fp32 12.6 against 18.1; but 64 x 1024 -> 16384, 1024 groups, 23 against 11);
    // fp32, whose tiles split their values first, up to two groups per CU (512 x 512 -> 1024 12.7 against 17.4, 768 rows 17.5 against 16.7).
    const dh_product& p = ps[0];
    if (n == 1 && p.a_by_reduction && p.b_by_reduction && !p.reduce_batch && !p.a_sum) {
        const int64_t groups = (int64_t)((p.J + 15) / 16) * p.batch, all = groups * ((p.I + THIN_ROWS - 1) / THIN_ROWS);
        if (p.I <= 32 ? groups >= CUS / 2 || (p.R <= 4096 && (int64_t)p.I * p.R <= 65536) : all <= (dtype == DH_F32 ? 2 : 1) * CUS && p.R <= 1024)
            return Shape{0, 16, 128, 1};
    }
    const bool split = dtype == DH_F32 && shortest >= 64;
    if (large < CUS && tile_steps < 16 * 2 * CUS) return Shape{64, 64, 128, split ? SPLIT : small <= 2 * CUS ? 4 : 2};
    if (split) return Shape{128, 128, 128, SPLIT};
    if (!aligned) return Shape{128, 128, 128, 1};
    if (dtype != DH_F32 && huge >= 2 * CUS && shortest >= 512 && held * 8 >= huge * 65536 * 7) return Shape{256, 256, 128, 2};
    return longest >= 1024 || large < CUS ? Shape{128, 128, 128, 2} : Shape{128, 128, 64, 3};
}

uint32_t at_least_1(int v) { return v > 0 ? (uint32_t)v : 1u; }

int cut(const dh_product* ps, int n, int dtype, Launch* L, float* ws, size_t* ws_bytes, bool* aligned, Shape* shape)
{
    const int64_t ch = dtype == DH_F32 ? 4 : 8, size = dtype == DH_F32 ? 4 : 2;
    // One kernel serves a launch, so one operand that is not aligned takes all of its products off the copying kernels: of a 16-bit head's
    // image sizes, only multiples of 128 px have levels of whole 16-byte rows everywhere (batch 64, fp16, us per MB forward / with all
    // gradients: 640 px 0.25 / 0.82, 768 px 0.29 / 0.82; 416 px 0.41 / 1.24, 576 px 0.35 / 1.13, 608 px 0.36 / 1.13, 800 px 0.41 / 1.17).
    *aligned = true;
    for (int w = 0; w < n; ++w) {
        const dh_product& p = ps[w];
        const int64_t all = p.lda | p.ldb | p.a_batch | p.b_batch;
        const int64_t ea = p.a_by_reduction ? p.R : p.I, eb = p.b_by_reduction ? p.R : p.J;
        if (all % ch || ea % ch || eb % ch || !dh_aligned16(p.a) || !dh_aligned16(p.b)) *aligned = false;
        if ((p.lda > p.ldb ? p.lda : p.ldb) >= (1ll << 31) / (256 * size)) *aligned = false;       // offsets in a tile are 32 bits
    }
    const Shape t = shape_of(ps, n, dtype, *aligned);
    const int64_t br = t.br / size;
    *shape = t;
    // Results that no cache could hold for their reader (32 MB of L2 in all) are stored past them.
    int64_t written = 0;
    for (int w = 0; w < n; ++w) written += (int64_t)ps[w].I * ps[w].J * (ps[w].reduce_batch ? 1 : ps[w].batch) * size * (ps[w].z ? 2 : 1);
    const bool large = written > (32ll << 20);
    int64_t total = 0;
    size_t bytes = 0;
    int64_t all_tiles = 0, tile_steps = 0;
    bool brief = true;                      // no reduction of more than 2 KB of a row
    for (int w = 0; w < n && t.bi; ++w) {
        const dh_product& p = ps[w];
        brief = brief && p.R * size * (p.reduce_batch ? p.batch : 1) <= 2048;
        const int64_t tiles = (int64_t)((p.I + t.bi - 1) / t.bi) * ((p.J + t.bj - 1) / t.bj) * (p.reduce_batch ? 1 : p.batch);
        all_tiles += tiles;
        tile_steps += tiles * ((p.R + br - 1) / br) * (p.reduce_batch ? p.batch : 1);
    }
    // Tiles for three quarters of the CUs to all of them, without the ring of the aligned kernels: two groups of waves in one workgroup
    // share a tile's reduction and join in LDS (1023 x 777 -> 1001 fp32: 24 us against 30 alone and 29 cut and joined by a launch; but
    // 128 x 4096 -> 4096, 128 tiles: 85 against 47).
    const bool grouped = t.bi == 64 && all_tiles <= CUS && all_tiles >= CUS * 3 / 4 && (!*aligned || t.stages == SPLIT);
    if (grouped) shape->groups = 2;
    // Fewer tiles than CUs: reductions are cut so that every workgroup of the launch has about the same number of steps, two
    // workgroups per CU.  Joining costs a launch and two passes over the partial sums, so at least 1 KB of a row each (1024^3 bf16, 256
    // tiles of 64 x 64, uncut: 11 us against 17), and nothing is cut that the deep ring passes in 16 steps (33 x 1024 -> 4096 9.3 against
    // 10.2, 1024 x 1000 -> 777 10.2 against 15.1; in 32 steps 33 x 2048 -> 512 12.6 against 10.6).  The same holds for operands of any
    // alignment, which have no ring but as short a reduction (256 x 777 -> 1501 11.6 against 12.6, 300 x 1023 -> 2001 13.8 against 16.2,
    // 601 channels at 1401 x 320 9.5 against 11.8; 1024 -> 255 channels of 13 x 13 cells 12.2 against 11.8).
    // About as many tiles as CUs are cut too where the reduction is long: one workgroup of a CU has nothing beside it while it waits
    // (4096 x 1024 over 8192 rows, 256 tiles of 128 x 128: bf16 78 us against 102, fp32 377 against 544).
    const int64_t once = 2 * CUS;
    int64_t each = (tile_steps + once - 1) / once;
    const bool cutting = t.bi && !grouped && !(brief && t.stages == 4) &&
                         (all_tiles < CUS || (t.bi == 128 && all_tiles <= CUS * 5 / 4 && each >= 4096 / t.br));
    if (each < 1024 / t.br) each = 1024 / t.br;
    int order[DH_MAX_PRODUCTS];
    for (int w = 0; w < n; ++w) {          // long reductions first: their workgroups are the ones a launch waits for
        int k = w;
        for (; k > 0 && ps[order[k - 1]].R < ps[w].R; --k) order[k] = order[k - 1];
        order[k] = w;
    }
    for (int w = 0; w < n; ++w) {
        const dh_product& p = ps[order[w]];
        Plan& q = L->plan[w];
        q.p = p;
        q.tiles_i = t.bi ? (p.I + t.bi - 1) / t.bi : (p.I + THIN_ROWS - 1) / THIN_ROWS;
        q.tiles_j = (p.J + t.bj - 1) / t.bj;
        q.batch_steps = (int)((p.R + br - 1) / br);
        const int64_t steps = (int64_t)q.batch_steps * (p.reduce_batch ? p.batch : 1);
        q.out_batches = p.reduce_batch ? 1 : p.batch;
        const int64_t tiles = (int64_t)q.tiles_i * q.tiles_j * q.out_batches;
        if (steps >= (1ll << 31) || tiles >= (1ll << 28) || (int64_t)q.tiles_i * q.tiles_j >= (1ll << 27)) return DH_ERR_ARG;
        q.steps = (int)steps;
        int64_t split = 1;
        if (cutting && tiles) split = (steps + each - 1) / each;
        if (split < 1) split = 1;
        q.per = (int)((steps + split - 1) / split);
        q.split = q.per ? (int)((steps + q.per - 1) / q.per) : 1;
        q.stream = large && p.ldo % ch == 0 && p.o_batch % ch == 0 && dh_aligned16(p.out) && dh_aligned16(p.z);
        q.partial = nullptr;
        if (q.split > 1) {
            q.partial = (float*)((char*)ws + bytes);
            bytes += ((size_t)q.split * q.out_batches * p.I * p.J * sizeof(float) + 255) & ~(size_t)255;
            q.partial_sum = (float*)((char*)ws + bytes);
            if (p.a_sum) bytes += ((size_t)q.split * p.I * sizeof(float) + 255) & ~(size_t)255;
        }
        L->first[w] = (int)total;
        q.count = (int)(tiles * q.split);
        q.by_plane = dh_make_fastdiv(at_least_1(q.tiles_i * q.tiles_j));
        q.by_group = dh_make_fastdiv(at_least_1(8 * q.tiles_j));
        q.by_tail = dh_make_fastdiv(at_least_1(q.tiles_i % 8));
        q.by_batches = dh_make_fastdiv(at_least_1(q.out_batches));
        total += (tiles * q.split + 7) / 8 * 8;
        if (total >= (1ll << 30)) return DH_ERR_ARG;
    }
    L->n = n;
    L->total = (int)total;
    *ws_bytes = bytes;
    return DH_OK;
}

int check(const dh_product* ps, int n, int dtype, int activation)
{
    if (!ps || n < 1 || n > DH_MAX_PRODUCTS || dtype < DH_F32 || dtype > DH_BF16 || activation < 0 || activation > DH_ACT_LAST)
        return DH_ERR_ARG;
    const uintptr_t esize = dtype == DH_F32 ? 4 : 2;
    for (int w = 0; w < n; ++w) {
        const dh_product& p = ps[w];
        if (p.I < 0 || p.J < 0 || p.R < 0 || p.batch < 0 || p.lda < 0 || p.ldb < 0 || p.ldo < 0 || p.ldr < 0) return DH_ERR_ARG;
        if (p.a_batch < 0 || p.b_batch < 0 || p.o_batch < 0 || p.res_batch < 0) return DH_ERR_ARG;
        if (p.I > DH_MAX_EXTENT || p.J > DH_MAX_EXTENT || p.R > DH_MAX_EXTENT) return DH_ERR_ARG;      // the last tile's end is an int
        if (!!p.a_by_reduction != !!ps[0].a_by_reduction || !!p.b_by_reduction != !!ps[0].b_by_reduction) return DH_ERR_ARG;
        if (!p.a_by_reduction && p.b_by_reduction) return DH_ERR_ARG;      // no caller has that pair
        const bool work = p.I > 0 && p.J > 0 && (p.reduce_batch || p.batch > 0);
        if (work && !p.out) return DH_ERR_ARG;
        if (p.a_sum && ((!p.reduce_batch && p.batch != 1) || p.J < 1)) return DH_ERR_ARG;
        if (work && p.R > 0 && p.batch > 0 && (!p.a || !p.b)) return DH_ERR_ARG;
        const uintptr_t all = (uintptr_t)p.a | (uintptr_t)p.b | (uintptr_t)p.out | (uintptr_t)p.z | (uintptr_t)p.residual | (uintptr_t)p.bias | (uintptr_t)p.a_sum;
        if (all % esize) return DH_ERR_ALIGN;
    }
    return DH_OK;
}

}  // namespace

extern "C" size_t dh_products_workspace(const dh_product* products, int n, int dtype)
{
    if (check(products, n, dtype, 0) != DH_OK) return 0;
    Launch L;
    size_t bytes = 0;
    bool aligned;
    Shape shape;
    return cut(products, n, dtype, &L, nullptr, &bytes, &aligned, &shape) == DH_OK ? bytes : 0;
}

extern "C" int dh_products(const dh_product* products, int n, int dtype, int activation, void* workspace, size_t workspace_bytes,
                           void* stream)
{
    int rc = check(products, n, dtype, activation);
    if (rc != DH_OK) return rc;
    Launch L;
    size_t bytes = 0;
    bool aligned;
    Shape shape;
    rc = cut(products, n, dtype, &L, (float*)workspace, &bytes, &aligned, &shape);
    if (rc != DH_OK) return rc;
    if (bytes > workspace_bytes || (bytes && !workspace)) return DH_ERR_WORKSPACE;
    if (bytes && !dh_aligned16(workspace)) return DH_ERR_ALIGN;
    L.act = activation;
    const bool arc = products[0].a_by_reduction != 0, brc = products[0].b_by_reduction != 0;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == DH_F32) return launch<float>(L, arc, brc, aligned, shape, st);
    if (dtype == DH_F16) return launch<_Float16>(L, arc, brc, aligned, shape, st);
    return launch<__bf16>(L, arc, brc, aligned, shape, st);
}

extern "C" size_t dh_product_slope_workspace(int64_t n) { return n > 0 ? (size_t)n * BIAS_SPLIT * sizeof(float) : 0; }

extern "C" int dh_product_slope(const void* dy, const void* z, void* dz, void* dbias, int64_t outer, int64_t n, int64_t inner,
                                int activation, int dtype, void* workspace, size_t workspace_bytes, void* stream)
{
    if (outer < 0 || n < 0 || inner < 0 || dtype < DH_F32 || dtype > DH_BF16 || activation < 0 || activation > DH_ACT_LAST) return DH_ERR_ARG;
    if (n == 0 || (!z && !dbias)) return DH_OK;
    if (n >= (1ll << 24) || outer >= (1ll << 40) || inner >= (1ll << 40)) return DH_ERR_ARG;
    int64_t per, all;
    if (__builtin_mul_overflow(outer, inner, &per) || __builtin_mul_overflow(per, n, &all) || all >= (1ll << 60)) return DH_ERR_ARG;
    if (per == 0 && !dbias) return DH_OK;
    if (per > 0 && (!dy || (z && !dz))) return DH_ERR_ARG;
    if (dbias && (!workspace || workspace_bytes < dh_product_slope_workspace(n))) return DH_ERR_WORKSPACE;
    if (dbias && !dh_aligned16(workspace)) return DH_ERR_ALIGN;
    if (((uintptr_t)dy | (uintptr_t)z | (uintptr_t)dz | (uintptr_t)dbias) % (dtype == DH_F32 ? 4 : 2)) return DH_ERR_ALIGN;
    hipStream_t st = (hipStream_t)stream;
    float* ws = (float*)workspace;
    if (dtype == DH_F32) return launch_slope<float>(dy, z, dz, dbias, outer, n, inner, activation, ws, st);
    if (dtype == DH_F16) return launch_slope<_Float16>(dy, z, dz, dbias, outer, n, inner, activation, ws, st);
    return launch_slope<__bf16>(dy, z, dz, dbias, outer, n, inner, activation, ws, st);
}
