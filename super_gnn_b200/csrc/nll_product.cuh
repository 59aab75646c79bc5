// The three matrix products of the many-class loss on the tensor cores (see linear_nll.cu):
//
//     logits   z[i, c]  = sum_k x[i, k] W[c, k]     epilogue: running (max, sum) of a row, or the gradient G
//     rows     gx[i, k] = sum_c G[i, c] W[c, k]
//     weights  gw[c, k] = sum_i G[i, c] x[i, k]
//
// The two gradients run as one launch where they are short: one tail, and one launch less to wait for.  Long ones run better
// alone (16k x 64k x 512 bf16: 4.37 ms against 4.65), where which of the two it is is known to the compiler and G has one reader
// at a time.
//
// One persistent block an SM.  A warp feeds operand tiles by TMA through a ring of shared memory buffers, a thread issues
// the tcgen05 products into tensor memory, eight warps turn finished 128 x 256 results into the outputs.  Two blocks of a
// cluster share a 256 x 256 result where that is faster (nll_in_pairs in linear_nll.cu): each brings 128 rows of the
// first operand and half of the second, 32 KB a step of 64 for 128 x 256 results where a block alone needs 48 KB.  The
// operands lie as their matrices do: x and W are read along k by the first product and across it by the other two, G along
// the classes by the second and across by the third, so that nothing is ever transposed in memory.
//
// fp32 operands come as two fp16 planes (v 2^e = v0 + v1, 22 bits; see linear_nll.cu) and three products
// v0 w0 + v0 w1 + v1 w0 a tile; bf16 operands as one plane and one product.  Tensor memory rounds every addition towards
// zero, a relative 2^-25 on average, and most of G has one sign: in the two gradients, whose reductions are long, the
// cross products of the planes, 2^-11 of the others, have sums of their own, and the main sums move on into registers every
// 512 of the reduction.  A sum over 55k classes would else be 5e-6 of itself too small (0.7e-6 so).
#pragma once
#include "umma.cuh"

namespace sgnn {

constexpr int kPM = 128, kPN = 256, kPK = 64;  // tile of a product, step of its reduction
constexpr int kPEpilogueWarps = 8;
constexpr int kPThreads = (kPEpilogueWarps + 2) * 32;
constexpr int kPWindow = 8;     // fp32 gradients: steps after which the main sums move on into registers
constexpr int kPAccCols = 512;  // all of the tensor memory: two results, or one and its cross products

// kLong...: the logits of fp32 operands over many features, with sums of their own for the cross products (see nll_logits_long)
enum ProductKind { kLogitStats, kLogitGrad, kGradients, kRowGrad, kWeightGrad, kLongStats, kLongGrad };
constexpr bool nll_is_stats(int kind) { return kind == kLogitStats || kind == kLongStats; }
constexpr bool nll_is_grad(int kind) { return kind == kLogitGrad || kind == kLongGrad; }
constexpr bool nll_is_logits(int kind) { return nll_is_stats(kind) || nll_is_grad(kind); }
constexpr bool nll_is_long(int kind) { return kind == kLongStats || kind == kLongGrad; }

struct ProductCall {
    CUtensorMap a, b, o;  // operands, result
    const int *total;     // rows in the loss
    int *failed;          // set when a wait gave up
    int row0, row_cap;    // this chunk of them
    int cls0, cls_count;  // this piece of the classes
    int feats;            // K
    int splits;           // of the reduction
    bool bf16;
    // logits
    const float *bias2;      // [classes rounded up to 256]: bias log2(e), -inf beyond the last class
    const float *row_scale;  // fp32: 2^-e of the rows of x (all of them) and of W
    const float *cls_scale;
    float2 *stats;           // [2 x class tiles, row_cap]: (maximum, sum of 2^(t - maximum)), in units of log2
    const float *lse2;       // [row_cap]
    float *picked2;          // [row_cap] the label's logit, from the same sums as the others
    const int *label;        // [row_cap]
    float *bias_part;        // [row_cap / 32, grad_ld]: sums of G over 32 rows, or nullptr
    int64_t grad_ld;
    // gradients of rows: o = [splits, row_cap, K rounded up to 32] fp32
    bool add;                // onto what the pieces (chunks) before have left there
    // gradients of weights: o = [splits, C, K rounded up to 32] fp32, or the result itself where nothing is left to add
    bool direct, direct_bf16;
    const unsigned *col_largest;  // fp32: the columns of x are scaled by it
    float scale;
    int64_t classes;
};

template <int PLANES, int CTAS>
struct ProductShared {
    static constexpr int kStages = (CTAS == 2 ? 6 : 4) / PLANES;
    static constexpr int kA = kPM * kPK * 2, kB = kPN / CTAS * kPK * 2;
    static constexpr int kStageBytes = PLANES * (kA + kB);
    static constexpr int kBox = 4096;  // result box of a warp: 32 rows of 128 bytes
};

template <int KIND, int PLANES, int CTAS>
constexpr int product_shared_bytes()
{
    using S = ProductShared<PLANES, CTAS>;
    const int ring = S::kStages * S::kStageBytes;
    if (nll_is_stats(KIND)) return ring + 2 * kPN * 8 + 256;
    if (nll_is_grad(KIND)) return ring + kPEpilogueWarps * S::kBox + kPN * 8 + 256;
    return ring + kPEpilogueWarps * S::kBox + 256;
}

// sizes of the product of this chunk and piece, from the number of rows in the loss
struct ProductUnits {
    int m, n, blocks, per_split, tiles_m, tiles_n, units, rows;
};

// `weights`: of the two gradients the second
template <int KIND, int CTAS>
__device__ __forceinline__ ProductUnits product_units(const ProductCall &c, bool weights)
{
    ProductUnits u;
    int rows = *c.total - c.row0;
    rows = rows < 0 ? 0 : rows < c.row_cap ? rows : c.row_cap;
    u.rows = rows;
    int red;
    if (nll_is_logits(KIND)) u.m = rows, u.n = c.cls_count, red = c.feats;
    else if (!weights) u.m = rows, u.n = c.feats, red = c.cls_count;
    else u.m = c.cls_count, u.n = c.feats, red = rows;
    u.blocks = (red + kPK - 1) / kPK;
    u.per_split = (u.blocks + c.splits - 1) / c.splits;
    u.tiles_m = (u.m + kPM * CTAS - 1) / (kPM * CTAS);
    u.tiles_n = (u.n + kPN - 1) / kPN;
    u.units = u.tiles_m * u.tiles_n * c.splits;
    return u;
}

// unit -> tile and range of reduction steps; an empty range still writes its zeros
struct ProductUnit {
    int m0, n0, split, first, count;  // m0: this block's first row
};
// Logits: the row tiles of one tile of classes follow each other (its part of W stays in L2).  Gradients: the column tiles of the
// same rows, which read the same part of G, the largest operand, at about the same time.
template <int KIND, int CTAS>
__device__ __forceinline__ ProductUnit product_unit(const ProductUnits &u, int i, int rank)
{
    constexpr bool kRowsFirst = nll_is_logits(KIND);
    ProductUnit t;
    const int tiles = u.tiles_m * u.tiles_n, in = i % tiles;
    const int tm = kRowsFirst ? in % u.tiles_m : in / u.tiles_n, tn = kRowsFirst ? in / u.tiles_m : in % u.tiles_n;
    t.m0 = (tm * CTAS + rank) * kPM, t.n0 = tn * kPN, t.split = i / tiles;
    t.first = t.split * u.per_split;
    const int end = t.first + u.per_split < u.blocks ? t.first + u.per_split : u.blocks;
    t.count = end > t.first ? end - t.first : 0;
    return t;
}

template <class T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float lo, float hi)
{
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack16<__half>(float lo, float hi)
{
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}

// 2^e that brings `largest` into [2^14, 2^15), and 2^-e; 1 for nothing but zeros and for what is not finite
__device__ __forceinline__ void plane_scale(float largest, float &up, float &down)
{
    up = down = 1.0f;
    if (!(largest > 0.f) || !(largest <= 3.402823466e+38f)) return;
    int e = 14 - ((int)(__float_as_uint(largest) >> 23) - 127);
    e = e < -126 ? -126 : e > 126 ? 126 : e;
    up = __uint_as_float((unsigned)(e + 127) << 23);
    down = __uint_as_float((unsigned)(127 - e) << 23);
}

constexpr float kGradScale = 32768.0f;  // fp16 planes of G: |G| <= 1 fills the range
// What the first plane of an operand of the gradients leaves, at most half of its last step, goes into the second one 2^11 times as
// large; the sums of the cross products are scaled back once.  Two planes then keep 22 bits of every value that is not below 2^-27
// of the largest (G, where 1 is known to be the largest: 2^-28), and are an absolute 2^-50 of the largest (2^-51) off below that.
// Unscaled these are 2^-16 and 2^-39 (2^-17 and 2^-40): a class of probability 2^-30 would keep 9 bits of its weights' gradient.
// The logits add both kinds of products into one sum and stay unscaled; there the scale is a row's own, and what is that small
// beside the row's largest value moves no logit.
constexpr float kSecondPlane = 2048.0f;

// `c`: the logits or the rows' gradient; `c2`: the weights' gradient (a kernel of one kind takes the same for both)
template <int KIND, int PLANES, int CTAS>
__global__ void __launch_bounds__(kPThreads, 1)
nll_product_kernel(const __grid_constant__ ProductCall c, const __grid_constant__ ProductCall c2)
{
    using S = ProductShared<PLANES, CTAS>;
    constexpr bool kLogits = nll_is_logits(KIND), kStats = nll_is_stats(KIND);
    constexpr bool kBmn = !kLogits;
    constexpr bool kCross = (!kLogits || nll_is_long(KIND)) && PLANES == 2;  // cross products have their own sums, in the other half of the tensor memory
    constexpr int kAcc = kCross ? 1 : 2;              // results in flight
    extern __shared__ __align__(1024) uint8_t base[];
    uint8_t *boxes = base + S::kStages * S::kStageBytes;
    uint8_t *after = boxes + (kStats ? 0 : kPEpilogueWarps * S::kBox);
    float *column = reinterpret_cast<float *>(after);  // logits: bias, then scale, of the classes of a tile
    constexpr int kColumns = kStats && kAcc == 2 ? 2 : 1;  // tiles whose classes are held at once
    uint8_t *behind = after + (kLogits ? kColumns * kPN * 8 : 0);
    uint64_t *full = reinterpret_cast<uint64_t *>(behind);
    uint64_t *empty = full + S::kStages, *acc_full = empty + S::kStages, *acc_empty = acc_full + 2;
    uint64_t *drained = acc_empty + 2;
    uint32_t *slot = reinterpret_cast<uint32_t *>(drained + 1);
    volatile int *gone = reinterpret_cast<volatile int *>(slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = CTAS == 2 ? (int)cluster_rank() : 0, first_unit = blockIdx.x / CTAS, unit_step = gridDim.x / CTAS;
    let_next_kernel_start();
    if ((smem_addr(base) & 1023u) != 0) {  // the swizzle counts from 1024-byte boundaries
        wait_for_kernels_before();
        if (threadIdx.x == 0) atomicExch(c.failed, 1);
        return;
    }

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) bar_init(full + s, 1), bar_init(empty + s, 1);
        for (int s = 0; s < 2; ++s) bar_init(acc_full + s, 1), bar_init(acc_empty + s, kPEpilogueWarps * CTAS);
        bar_init(drained, 1);
        *gone = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kPEpilogueWarps + 1) {
        if (CTAS == 2) tmem_alloc_pair(slot, kPAccCols);
        else tmem_alloc(slot, kPAccCols);
    }
    tc_fence_before();
    __syncthreads();
    if (CTAS == 2) cluster_sync();  // the barriers of both blocks are there
    tc_fence_after();
    const uint32_t tmem = *slot;
    wait_for_kernels_before();
    constexpr bool kBoth = KIND == kGradients;
    const ProductUnits u1 = product_units<KIND, CTAS>(c, KIND == kWeightGrad), u2 = kBoth ? product_units<KIND, CTAS>(c2, true) : u1;
    const int units = u1.units + (kBoth ? u2.units : 0);

    if (warp == kPEpilogueWarps) {
        // ---- loads ----
        if (lane == 0) {
            tma_prefetch(&c.a);
            tma_prefetch(&c.b);
            if (kBoth) tma_prefetch(&c2.a), tma_prefetch(&c2.b);
            int stage = 0;
            unsigned phase = 0, used = 0;
            bool ok = true;
            for (int i = first_unit; i < units && ok; i += unit_step) {
                const bool second = kBoth && i >= u1.units, weights = KIND == kWeightGrad || second;
                const ProductUnits &u = second ? u2 : u1;
                const CUtensorMap *ma = second ? &c2.a : &c.a, *mb = second ? &c2.b : &c.b;
                const ProductUnit t = product_unit<KIND, CTAS>(u, second ? i - u1.units : i, rank);
                const int left = u.n - t.n0, own_n = (left < kPN ? (left + 15) / 16 * 16 : kPN) / CTAS;  // columns of the second operand here
                const int runs = kBmn ? (own_n + 63) / 64 : 1;
                const unsigned bytes = PLANES * (S::kA + (kBmn ? runs * 64 * kPK * 2 : S::kB));
                for (int k = 0; k < t.count; ++k) {
                    ok = bar_wait(empty + stage, phase ^ 1, gone);
                    if (!ok) break;
                    uint8_t *at = base + stage * S::kStageBytes;
                    if (rank == 0) bar_expect(full + stage, CTAS * bytes);
                    const uint32_t lead = CTAS == 2 ? leader_addr(full + stage) : 0u;
                    const auto load = [&](void *dst, const CUtensorMap *map, int x, int y, int z) {
                        if (CTAS == 2) tma_load_pair(dst, map, x, y, z, lead);
                        else tma_load(dst, map, x, y, z, full + stage);
                    };
                    const int k0 = (t.first + k) * kPK;
#pragma unroll
                    for (int p = 0; p < PLANES; ++p) {
                        uint8_t *pa = at + p * S::kA, *pb = at + PLANES * S::kA + p * S::kB;
                        if (weights) {
                            load(pa, ma, t.m0, k0, p);
                            load(pa + 64 * kPK * 2, ma, t.m0 + 64, k0, p);
                        } else {
                            load(pa, ma, k0, t.m0 + (kLogits ? c.row0 : 0), p);
                        }
                        if (kBmn) {
                            const int k1 = k0 + (weights ? c.row0 : c.cls0);
                            for (int r = 0; r < runs; ++r) load(pb + r * 64 * kPK * 2, mb, t.n0 + rank * own_n + 64 * r, k1, p);
                        } else {
                            load(pb, mb, k0, t.n0 + c.cls0 + rank * (kPN / CTAS), p);
                        }
                    }
                    ++used;
                    if (++stage == S::kStages) stage = 0, phase ^= 1;
                }
            }
            if (!ok) {  // copies of this block still under way: their buffers must not be left to another block
                if (rank != 0) {  // what counts them is the other block's
                    const uint64_t until = now_ns() + kWaitNs / 8;
                    while (now_ns() < until) __nanosleep(1000);
                }
                if (rank == 0) ring_drain(full, used, S::kStages);
            }
        }
        __syncwarp();
    } else if (warp == kPEpilogueWarps + 1) {
        // ---- products (of both blocks: the first one's) ----
        if (lane == 0 && rank == 0) {
            int stage = 0, acc = 0;
            unsigned phase = 0, acc_phase = 0;
            bool ok = true;
            const auto commit = [&](uint64_t *bar) {
                if (CTAS == 2) tc_commit_pair(bar);
                else tc_commit(bar);
            };
            const auto product = [&](uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
                if (CTAS == 2) umma_pair(d, a, b, idesc, add);
                else umma(d, a, b, idesc, add);
            };
            for (int i = first_unit; i < units && ok; i += unit_step) {
                const bool second = kBoth && i >= u1.units, weights = KIND == kWeightGrad || second;
                const ProductUnits &u = second ? u2 : u1;
                const ProductUnit t = product_unit<KIND, CTAS>(u, second ? i - u1.units : i, rank);
                const int left = u.n - t.n0;
                const int n = kBmn ? (left < kPN ? (left + 15) / 16 * 16 : kPN) : kPN;
                const uint32_t idesc = umma_idesc(c.bf16, weights, kBmn, n, kPM * CTAS);
                ok = bar_wait(acc_empty + acc, acc_phase ^ 1, gone);
                if (!ok) break;
                tc_fence_after();
                const uint32_t d = tmem + acc * kPN;
                for (int k = 0; k < t.count; ++k) {
                    ok = bar_wait(full + stage, phase, gone);
                    if (!ok) break;
                    tc_fence_after();
                    const bool starts = kCross && k % kPWindow == 0, ends = kCross && k % kPWindow == kPWindow - 1 && k + 1 < t.count;
                    const uint8_t *at = base + stage * S::kStageBytes;
                    // eight-row groups 1024 bytes apart; MN-major operands: 64-element runs of kPK rows each
                    const unsigned a_run = weights ? 64 * kPK * 2 : 16, b_run = kBmn ? 64 * kPK * 2 : 16;
                    uint64_t da[PLANES], db[PLANES];
#pragma unroll
                    for (int p = 0; p < PLANES; ++p) {
                        da[p] = umma_desc(at + p * S::kA, a_run, 1024);
                        db[p] = umma_desc(at + PLANES * S::kA + p * S::kB, b_run, 1024);
                    }
                    // sixteen steps of the reduction: 32 bytes along a row, or two groups of eight rows
                    const uint64_t step_a = (weights ? 2048u : 32u) >> 4, step_b = (kBmn ? 2048u : 32u) >> 4;
                    const auto main = [&](int j) { product(d, da[0] + step_a * j, db[0] + step_b * j, idesc, kCross ? !starts || j > 0 : k > 0 || j > 0); };
                    const auto cross = [&](int j) {
                        const uint32_t dx = kCross ? tmem + kPN : d;
                        product(dx, da[0] + step_a * j, db[PLANES - 1] + step_b * j, idesc, !kCross || k > 0 || j > 0);
                        product(dx, da[PLANES - 1] + step_a * j, db[0] + step_b * j, idesc, true);
                    };
                    if (kCross) {  // the cross products run while the main sums are read
                        if (starts && k > 0) {
#pragma unroll
                            for (int j = 0; j < kPK / 16; ++j) cross(j);
                            ok = bar_wait(acc_empty, acc_phase ^ 1, gone);
                            if (!ok) break;
                            tc_fence_after();
                        }
#pragma unroll
                        for (int j = 0; j < kPK / 16; ++j) main(j);
                        if (ends) commit(acc_full), acc_phase ^= 1;
                        if (!starts || k == 0) {
#pragma unroll
                            for (int j = 0; j < kPK / 16; ++j) cross(j);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < kPK / 16; ++j) {
                            main(j);
                            if (PLANES == 2) cross(j);
                        }
                    }
                    commit(empty + stage);
                    if (++stage == S::kStages) stage = 0, phase ^= 1;
                }
                if (!ok) break;
                commit(acc_full + acc);
                if (++acc == kAcc) acc = 0, acc_phase ^= 1;
            }
            if (!ok) {  // products still under way write tensor memory and read the buffers
                commit(drained);
                bar_drain(drained, 0);
            }
        }
        __syncwarp();
    } else {
        // ---- results ----
        const int quarter = warp & 3, half = warp >> 2, tid = threadIdx.x;
        uint8_t *box = boxes + warp * S::kBox;
        uint8_t *box_row = box + lane * 128;
        int acc = 0;
        unsigned acc_phase = 0;
        for (int i = first_unit; i < units; i += unit_step) {
            const bool second = kBoth && i >= u1.units, weights = KIND == kWeightGrad || second;
            const ProductUnits &u = second ? u2 : u1;
            const ProductUnit t = product_unit<KIND, CTAS>(u, second ? i - u1.units : i, rank);
            const int row = t.m0 + quarter * 32 + lane;  // of the product
            float *bias_col = column + (kColumns == 2 ? acc : 0) * 2 * kPN, *scale_col = bias_col + kPN;
            if (kLogits) {
                const int cls = c.cls0 + t.n0 + tid;  // the arrays cover whole tiles
                const float b = __ldg(c.bias2 + cls);
                if (kColumns == 1) asm volatile("bar.sync 1, %0;" ::"n"(kPEpilogueWarps * 32) : "memory");
                bias_col[tid] = b;
                if (PLANES == 2) scale_col[tid] = __ldg(c.cls_scale + cls);
                asm volatile("bar.sync 1, %0;" ::"n"(kPEpilogueWarps * 32) : "memory");
            }
            float scale = 1.4426950408889634f, lse2 = 0.f;
            if (kLogits && PLANES == 2) scale *= __ldg(c.row_scale + c.row0 + (row < u.m ? row : 0));
            if (nll_is_grad(KIND) && row < u.m) lse2 = __ldg(c.lse2 + row);
            float sum[kCross ? 4 : 1][32];  // the main sums of the windows before the last
            if constexpr (kCross) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 32; ++e) sum[j][e] = 0.f;
#pragma unroll 1
                for (int k = kPWindow; k < t.count; k += kPWindow) {
                    if (!bar_wait(acc_full, acc_phase, gone)) break;
                    tc_fence_after();
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (t.n0 + half * 128 + 32 * j >= u.n) break;
                        float x[32];
                        tmem_load32(tmem + half * 128 + 32 * j + ((uint32_t)quarter << 21), x);
                        tmem_load_wait(x);
#pragma unroll
                        for (int e = 0; e < 32; ++e) sum[j][e] += x[e];
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if (CTAS == 2) leader_arrive(acc_empty);
                        else bar_arrive(acc_empty);
                    }
                    acc_phase ^= 1;
                }
            }
            if (!bar_wait(acc_full + acc, acc_phase, gone)) {  // the others may stand at the barrier above: keep coming to it
                if (++acc == kAcc) acc = 0, acc_phase ^= 1;
                continue;
            }
            tc_fence_after();
            const uint32_t d = tmem + acc * kPN + half * 128 + ((uint32_t)quarter << 21);
            const bool there = t.count > 0;  // an empty range of the reduction: zeros
            float v[32], ahead[32];
            if (kLogits && !kCross) tmem_load32(d, ahead);
            // logits in units of log2, 32 columns at a time; the next ones come while these are worked on (not beside the sums of the
            // windows before, which fill the registers)
            const auto logits = [&](int j) {
                if constexpr (kCross) {
                    tmem_load32(d + 32 * j, v);
                    tmem_load32(d + kPN + 32 * j, ahead);
                    tmem_load_wait(v);
                    tmem_load_wait(ahead);
#pragma unroll
                    for (int e = 0; e < 32; ++e) v[e] = (v[e] + sum[j][e]) + ahead[e];
                } else {
                    tmem_load_wait(ahead);
#pragma unroll
                    for (int e = 0; e < 32; ++e) v[e] = ahead[e];
                    if (j < 3) tmem_load32(d + 32 * (j + 1), ahead);
                }
                const float4 *b4 = reinterpret_cast<const float4 *>(bias_col + half * 128 + 32 * j);
                const float4 *s4 = reinterpret_cast<const float4 *>(scale_col + half * 128 + 32 * j);
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    const float4 b = b4[q];
                    if (PLANES == 2) {
                        const float4 w = s4[q];
                        v[4 * q] *= w.x, v[4 * q + 1] *= w.y, v[4 * q + 2] *= w.z, v[4 * q + 3] *= w.w;
                    }
                    v[4 * q] = __fmaf_rn(v[4 * q], scale, b.x), v[4 * q + 1] = __fmaf_rn(v[4 * q + 1], scale, b.y);
                    v[4 * q + 2] = __fmaf_rn(v[4 * q + 2], scale, b.z), v[4 * q + 3] = __fmaf_rn(v[4 * q + 3], scale, b.w);
                }
            };
            // the box is free again / filled: hand it on
            const auto box_free = [&]() {
                if (lane == 0) store_wait_read();
                __syncwarp();
            };
            const auto box_done = [&]() {
                async_fence();
                __syncwarp();
            };
            if constexpr (kStats) {
                float mx = -INFINITY, total = 0.f;
                const int label = row < u.m ? c.label[row] - c.cls0 - t.n0 - half * 128 : -1;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    logits(j);
                    const int at = label - 32 * j;
                    if (at >= 0 && at < 32) {  // in these columns
                        float z = v[0];
#pragma unroll
                        for (int e = 1; e < 32; ++e) z = e == at ? v[e] : z;
                        c.picked2[row] = z;
                    }
                    float top = mx;
#pragma unroll
                    for (int e = 0; e < 32; ++e) top = fmaxf(top, v[e]);
                    const float ref = top == -INFINITY ? 0.f : top;
                    total *= exp2_fast(mx - ref);
#pragma unroll
                    for (int e = 0; e < 32; ++e) total += exp2_fast(v[e] - ref);
                    mx = top;
                }
                if (row < u.m) c.stats[(int64_t)(t.n0 / 128 + half) * c.row_cap + row] = make_float2(mx, total);
            } else if constexpr (nll_is_grad(KIND)) {
                const int label = row < u.m ? c.label[row] - c.cls0 - t.n0 - half * 128 : -1;
                const float own = label >= 0 && label < 128  // G of the label's class, p - 1, without the cancellation of a p next to 1
                                      ? expm1f((__ldg(c.picked2 + row) - lse2) * 0.6931471805599453f) * (PLANES == 2 ? kGradScale : 1.0f)
                                      : 0.f;
                const int x0 = t.n0 + half * 128, y0 = t.m0 + quarter * 32;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    logits(j);
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        v[e] = row < u.m ? exp2_fast(v[e] - lse2) : 0.f;
                        if (PLANES == 2) v[e] *= kGradScale;
                    }
                    const int at = label - 32 * j;  // 0 .. 31: in these columns
                    float *part = c.bias_part + (int64_t)(y0 >> 5) * c.grad_ld + x0;
                    if (PLANES == 1) {  // 64 columns a box: 128 bytes a row, two turns
                        if ((j & 1) == 0) box_free();
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            uint4 w;
                            uint32_t *pw = reinterpret_cast<uint32_t *>(&w);
#pragma unroll
                            for (int e = 0; e < 4; ++e) pw[e] = pack16<__nv_bfloat16>(v[8 * q + 2 * e], v[8 * q + 2 * e + 1]);
                            const int place = ((j & 1) * 4 + q) ^ (lane & 7);
                            *reinterpret_cast<uint4 *>(box_row + place * 16) = w;
                        }
                        if (at >= 0 && at < 32) {
                            const int place = ((j & 1) * 4 + at / 8) ^ (lane & 7);
                            *reinterpret_cast<__nv_bfloat16 *>(box_row + place * 16 + at % 8 * 2) = __float2bfloat16_rn(own);
                        }
                        if (j & 1) {
                            box_done();
                            if (lane == 0 && y0 < c.row_cap) {
                                tma_store(&c.o, box, x0 + 32 * (j - 1), y0, 0);
                                store_commit();
                            }
                            if (c.bias_part != nullptr && y0 < c.row_cap) {  // two columns a lane, down the rows of the box
                                float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                                for (int r = 0; r < 32; ++r) {
                                    const uint32_t two = *reinterpret_cast<const uint32_t *>(box + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
                                    sum.x += __uint_as_float(two << 16), sum.y += __uint_as_float(two & 0xFFFF0000u);
                                }
                                *reinterpret_cast<float2 *>(part + 32 * (j - 1) + 2 * lane) = sum;
                            }
                        }
                    } else {  // 32 columns of both planes: 64 bytes a row each
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] = e == at ? own : v[e];
                        box_free();
                        uint8_t *r0 = box + lane * 64, *r1 = r0 + 2048;
                        const int turn = (lane >> 1) & 3;
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            uint4 w0, w1;
                            uint32_t *p0 = reinterpret_cast<uint32_t *>(&w0), *p1 = reinterpret_cast<uint32_t *>(&w1);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float g0 = v[8 * q + 2 * e], g1 = v[8 * q + 2 * e + 1];
                                p0[e] = pack16<__half>(g0, g1);
                                const float2 r = __half22float2(*reinterpret_cast<const __half2 *>(p0 + e));
                                p1[e] = pack16<__half>((g0 - r.x) * kSecondPlane, (g1 - r.y) * kSecondPlane);
                            }
                            *reinterpret_cast<uint4 *>(r0 + (q ^ turn) * 16) = w0;
                            *reinterpret_cast<uint4 *>(r1 + (q ^ turn) * 16) = w1;
                        }
                        box_done();
                        if (lane == 0 && y0 < c.row_cap) {
                            tma_store(&c.o, box, x0 + 32 * j, y0, 0);
                            tma_store(&c.o, box + 2048, x0 + 32 * j, y0, 1);
                            store_commit();
                        }
                        if (c.bias_part != nullptr && y0 < c.row_cap) {
                            // 32 rows x 32 columns: every exchange halves the columns a lane carries; lane l ends with column l
#pragma unroll
                            for (int o = 16; o > 0; o >>= 1) {
                                const bool upper = (lane & o) != 0;
#pragma unroll
                                for (int e = 0; e < o; ++e) {
                                    const float keep = upper ? v[e + o] : v[e], give = upper ? v[e] : v[e + o];
                                    v[e] = keep + __shfl_xor_sync(FULL, give, o);
                                }
                            }
                            part[32 * j + lane] = v[0];
                        }
                    }
                }
            } else {
                const bool direct = weights && c2.direct, wide = direct && c2.direct_bf16, add = weights ? c2.add : c.add;
                const CUtensorMap *mo = second ? &c2.o : &c.o;
                const int y0 = t.m0 + quarter * 32 + (weights ? c.cls0 : 0), end = weights ? (int)c.classes : c.row_cap;
#pragma unroll(kCross ? 4 : 1)
                for (int j = 0; j < 4; ++j) {
                    const int k0 = t.n0 + half * 128 + 32 * j;
                    if (k0 >= u.n) break;
                    tmem_load32(d + 32 * j, v);
                    tmem_load_wait(v);
                    if (kCross) {
                        float x[32];
                        tmem_load32(d + kPN + 32 * j, x);
                        tmem_load_wait(x);
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] = __fmaf_rn(x[e], 1.0f / kSecondPlane, v[e] + sum[j][e]);
                    }
                    if (!there) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] = 0.f;
                    }
                    if (direct) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] *= c2.scale;
                        if (PLANES == 2) {
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                float up, down;
                                plane_scale(__uint_as_float(k0 + e < u.n ? __ldg(c2.col_largest + k0 + e) : 0u), up, down);
                                v[e] *= down;
                            }
                        }
                    }
                    if (!wide || (j & 1) == 0) box_free();
                    if (!wide) {
#pragma unroll
                        for (int q = 0; q < 8; ++q)
                            *reinterpret_cast<float4 *>(box_row + (q ^ (lane & 7)) * 16) =
                                make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
                    } else {
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            uint4 w;
                            uint32_t *pw = reinterpret_cast<uint32_t *>(&w);
#pragma unroll
                            for (int e = 0; e < 4; ++e) pw[e] = pack16<__nv_bfloat16>(v[8 * q + 2 * e], v[8 * q + 2 * e + 1]);
                            *reinterpret_cast<uint4 *>(box_row + (((j & 1) * 4 + q) ^ (lane & 7)) * 16) = w;
                        }
                        if ((j & 1) == 0 && k0 + 32 < u.n) continue;  // 64 columns a box
                    }
                    box_done();
                    if (lane == 0 && y0 < end) {
                        const int x0 = wide ? t.n0 + half * 128 + 64 * (j >> 1) : k0;
                        if (add) tma_add(mo, box, x0, y0, t.split);
                        else tma_store(mo, box, x0, y0, t.split);
                        store_commit();
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (CTAS == 2) leader_arrive(acc_empty + acc);
                else bar_arrive(acc_empty + acc);
            }
            if (++acc == kAcc) acc = 0, acc_phase ^= 1;
        }
        if (!kStats && lane == 0) store_wait_all();
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (CTAS == 2) cluster_sync();  // nothing of the other block is under way to this one any more
    tc_fence_after();
    if (threadIdx.x == 0 && *gone) atomicExch(c.failed, 1);
    if (warp == kPEpilogueWarps + 1) {
        if (CTAS == 2) tmem_free_pair(tmem, kPAccCols);
        else tmem_free(tmem, kPAccCols);
    }
}

}  // namespace sgnn
