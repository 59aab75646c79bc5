// The three matrix products of the many-class loss on the tensor cores (see linear_nll.cu):
//
//     logits   z[i, c]  = sum_k x[i, k] W[c, k]     epilogue: running (max, sum) of a row, or the gradient G
//     rows     gx[i, k] = sum_c G[i, c] W[c, k]
//     weights  gw[c, k] = sum_i G[i, c] x[i, k]     and gb[c] = sum_i G[i, c], a product with ones
//
// One persistent block an SM.  A warp feeds 128 x 64 and 256 x 64 operand tiles by TMA through a ring of shared memory
// buffers, a thread issues the tcgen05 products into tensor memory, eight warps turn finished 128 x 256 results into
// the outputs.  The operands lie as their matrices do: x and W are read along k by the first product and across it by the
// other two, G along the classes by the second and across by the third, so that nothing is ever transposed in memory.
//
// fp32 operands come as two fp16 planes (v 2^e = v0 + v1, 22 bits; see split planes in linear_nll.cu) and three products
// v0 w0 + v0 w1 + v1 w0 a tile; bf16 operands as one plane and one product.
#pragma once
#include "umma.cuh"

namespace sgnn {

constexpr int kPM = 128, kPN = 256, kPK = 64;  // tile of a product, step of its reduction
constexpr int kPEpilogueWarps = 8;
constexpr int kPThreads = (kPEpilogueWarps + 2) * 32;
constexpr int kPAccCols = 512;  // all of the tensor memory: two results, or one and the sums of the bias gradient

enum ProductKind { kLogitStats, kLogitGrad, kRowGrad, kWeightGrad };

struct ProductCall {
    CUtensorMap a, b;
    const int *total;     // rows in the loss
    int *failed;          // set when a wait gave up
    int row0, row_cap;    // this chunk of them
    int cls0, cls_count;  // this piece of the classes
    int feats;            // K
    int splits;           // of the reduction
    bool bf16;
    // logits
    const float *bias2;      // [classes rounded up to 256]: bias log2(e), -inf beyond the last class
    const float *row_scale;  // fp32: 2^-e of the rows of x (all of them) and of W; nullptr: 1
    const float *cls_scale;
    float2 *stats;           // [2 x class tiles, row_cap]: (maximum, sum of 2^(t - maximum)), in units of log2
    const float *lse2;       // [row_cap]
    const float *picked2;    // [row_cap] the label's logit
    const int *label;        // [row_cap]
    uint16_t *grad;          // [planes, row_cap, grad_ld]
    int64_t grad_ld;
    // gradients
    float *out;           // rows: [splits, row_cap, out_ld]; weights: [splits, classes, out_ld] at the piece's first class
    int64_t out_ld, out_split;
    bool add;
    // weights, when nothing is left to add: the result itself
    void *gw;
    int64_t gw_ld;
    void *gb;
    bool gw_f32, gb_f32;
    const float *col_scale;  // fp32: 2^-e of the columns of x
    float scale;
    float *bias_out;  // [splits, classes] at the piece's first class
    int64_t bias_split;
};

template <int PLANES>
struct ProductShared {
    static constexpr int kStages = 4 / PLANES;
    static constexpr int kA = kPM * kPK * 2, kB = kPN * kPK * 2;
    static constexpr int kStageBytes = PLANES * (kA + kB);
    static constexpr int kOnes = 16 * kPK * 2;
    static constexpr int kBytes = kStages * kStageBytes + kOnes + 2 * kPN * 8 + 256 + 1024;
};

// sizes of the product of this chunk and piece, from the number of rows in the loss
struct ProductUnits {
    int m, n, blocks, per_split, tiles_m, tiles_n, units, rows;
};

template <int KIND>
__device__ __forceinline__ ProductUnits product_units(const ProductCall &c)
{
    ProductUnits u;
    int rows = *c.total - c.row0;
    rows = rows < 0 ? 0 : rows < c.row_cap ? rows : c.row_cap;
    u.rows = rows;
    int red;
    if (KIND == kLogitStats || KIND == kLogitGrad) u.m = rows, u.n = c.cls_count, red = c.feats;
    else if (KIND == kRowGrad) u.m = rows, u.n = c.feats, red = c.cls_count;
    else u.m = c.cls_count, u.n = c.feats, red = rows;
    u.blocks = (red + kPK - 1) / kPK;
    u.per_split = (u.blocks + c.splits - 1) / c.splits;
    u.tiles_m = (u.m + kPM - 1) / kPM;
    u.tiles_n = (u.n + kPN - 1) / kPN;
    u.units = u.tiles_m * u.tiles_n * c.splits;
    return u;
}

// unit -> tile and range of reduction steps; an empty range still writes its zeros
struct ProductUnit {
    int m0, n0, split, first, count;
};
__device__ __forceinline__ ProductUnit product_unit(const ProductUnits &u, int i)
{
    ProductUnit t;
    const int tm = i % u.tiles_m, rest = i / u.tiles_m;
    t.m0 = tm * kPM, t.n0 = rest % u.tiles_n * kPN, t.split = rest / u.tiles_n;
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

constexpr float kGradScale = 32768.0f;  // fp16 planes of G: |G| <= 1 fills the range, 2^-40 is the smallest step

template <int KIND, int PLANES>
__global__ void __launch_bounds__(kPThreads, 1) nll_product_kernel(const __grid_constant__ ProductCall c)
{
    using S = ProductShared<PLANES>;
    constexpr bool kLogits = KIND == kLogitStats || KIND == kLogitGrad;
    constexpr bool kAmn = KIND == kWeightGrad, kBmn = !kLogits;
    constexpr int kAcc = KIND == kWeightGrad ? 1 : 2;  // results in flight
    extern __shared__ uint8_t raw[];
    uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) / 1024 * 1024);
    uint8_t *ones = base + S::kStages * S::kStageBytes;
    float2 *column = reinterpret_cast<float2 *>(ones + S::kOnes);  // [2][256]: (bias, scale) of the classes of a tile
    uint64_t *full = reinterpret_cast<uint64_t *>(column + 2 * kPN);
    uint64_t *empty = full + S::kStages, *acc_full = empty + S::kStages, *acc_empty = acc_full + 2;
    uint64_t *drained = acc_empty + 2;
    uint32_t *slot = reinterpret_cast<uint32_t *>(drained + 1);
    volatile int *gone = reinterpret_cast<volatile int *>(slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const ProductUnits u = product_units<KIND>(c);
    if ((int)blockIdx.x >= u.units) return;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) bar_init(full + s, 1), bar_init(empty + s, 1);
        for (int s = 0; s < 2; ++s) bar_init(acc_full + s, 1), bar_init(acc_empty + s, kPEpilogueWarps);
        bar_init(drained, 1);
        *gone = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (KIND == kWeightGrad) {
        const uint32_t one = c.bf16 ? 0x3F803F80u : 0x3C003C00u;
        for (int i = threadIdx.x; i < S::kOnes / 4; i += kPThreads) reinterpret_cast<uint32_t *>(ones)[i] = one;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == kPEpilogueWarps + 1) tmem_alloc(slot, kPAccCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *slot;

    if (warp == kPEpilogueWarps) {
        // ---- loads ----
        if (lane == 0) {
            tma_prefetch(&c.a);
            tma_prefetch(&c.b);
            int stage = 0;
            unsigned phase = 0, used = 0;
            bool ok = true;
            for (int i = blockIdx.x; i < u.units && ok; i += gridDim.x) {
                const ProductUnit t = product_unit(u, i);
                const int runs = kBmn ? ((u.n - t.n0 < kPN ? u.n - t.n0 : kPN) + 63) / 64 : 1;
                const unsigned bytes = PLANES * (S::kA + (kBmn ? runs * 64 * kPK * 2 : S::kB));
                for (int k = 0; k < t.count; ++k) {
                    ok = bar_wait(empty + stage, phase ^ 1, gone);
                    if (!ok) break;
                    uint8_t *at = base + stage * S::kStageBytes;
                    bar_expect(full + stage, bytes);
                    const int k0 = (t.first + k) * kPK;
#pragma unroll
                    for (int p = 0; p < PLANES; ++p) {
                        uint8_t *pa = at + p * S::kA, *pb = at + PLANES * S::kA + p * S::kB;
                        if (kAmn) {
                            tma_load(pa, &c.a, t.m0, k0, p, full + stage);
                            tma_load(pa + 64 * kPK * 2, &c.a, t.m0 + 64, k0, p, full + stage);
                        } else {
                            tma_load(pa, &c.a, k0, t.m0 + (kLogits ? c.row0 : 0), p, full + stage);
                        }
                        if (kBmn) {
                            const int k1 = k0 + (KIND == kRowGrad ? c.cls0 : c.row0);
                            for (int r = 0; r < runs; ++r) tma_load(pb + r * 64 * kPK * 2, &c.b, t.n0 + 64 * r, k1, p, full + stage);
                        } else {
                            tma_load(pb, &c.b, k0, t.n0 + c.cls0, p, full + stage);
                        }
                    }
                    ++used;
                    if (++stage == S::kStages) stage = 0, phase ^= 1;
                }
            }
            if (!ok) {  // copies of this block still under way: their buffers must not be left to another block
                for (int s = 0; s < S::kStages; ++s) {
                    if (used < (unsigned)(s + 1)) continue;
                    const unsigned uses = (used - 1 - s) / S::kStages + 1;  // fills of this buffer so far
                    bar_drain(full + s, (uses - 1) & 1);
                }
            }
        }
        __syncwarp();
    } else if (warp == kPEpilogueWarps + 1) {
        // ---- products ----
        if (lane == 0) {
            int stage = 0, acc = 0;
            unsigned phase = 0, acc_phase = 0;
            bool ok = true;
            for (int i = blockIdx.x; i < u.units && ok; i += gridDim.x) {
                const ProductUnit t = product_unit(u, i);
                const int left = u.n - t.n0;
                const int n = kBmn ? (left < kPN ? (left + 15) / 16 * 16 : kPN) : kPN;
                const uint32_t idesc = umma_idesc(c.bf16, kAmn, kBmn, n), idesc_ones = umma_idesc(c.bf16, kAmn, false, 16);
                ok = bar_wait(acc_empty + acc, acc_phase ^ 1, gone);
                if (!ok) break;
                tc_fence_after();
                const uint32_t d = tmem + acc * kPN;
                for (int k = 0; k < t.count; ++k) {
                    ok = bar_wait(full + stage, phase, gone);
                    if (!ok) break;
                    tc_fence_after();
                    const uint8_t *at = base + stage * S::kStageBytes;
                    // eight-row groups 1024 bytes apart; MN-major operands: 64-element runs of kPK rows each
                    const unsigned a_run = kAmn ? 64 * kPK * 2 : 16, b_run = kBmn ? 64 * kPK * 2 : 16;
                    uint64_t da[PLANES], db[PLANES];
#pragma unroll
                    for (int p = 0; p < PLANES; ++p) {
                        da[p] = umma_desc(at + p * S::kA, a_run, 1024);
                        db[p] = umma_desc(at + PLANES * S::kA + p * S::kB, b_run, 1024);
                    }
                    const uint64_t dones = umma_desc(ones, 16, 1024);
#pragma unroll
                    for (int j = 0; j < kPK / 16; ++j) {
                        // sixteen steps of the reduction: 32 bytes along a row, or two groups of eight rows
                        const uint64_t sa = (kAmn ? 2048u : 32u) * j >> 4, sb = (kBmn ? 2048u : 32u) * j >> 4;
                        const bool more = k > 0 || j > 0;
                        umma(d, da[0] + sa, db[0] + sb, idesc, more);
                        if (PLANES == 2) {
                            umma(d, da[0] + sa, db[PLANES - 1] + sb, idesc, true);
                            umma(d, da[PLANES - 1] + sa, db[0] + sb, idesc, true);
                        }
                        if (KIND == kWeightGrad && t.n0 == 0) {
                            umma(tmem + kPN, da[0] + sa, dones, idesc_ones, more);
                            if (PLANES == 2) umma(tmem + kPN, da[PLANES - 1] + sa, dones, idesc_ones, true);
                        }
                    }
                    tc_commit(empty + stage);
                    if (++stage == S::kStages) stage = 0, phase ^= 1;
                }
                if (!ok) break;
                tc_commit(acc_full + acc);
                if (++acc == kAcc) acc = 0, acc_phase ^= 1;
            }
            if (!ok) {  // products still under way write tensor memory and read the buffers
                tc_commit(drained);
                bar_drain(drained, 0);
            }
        }
        __syncwarp();
    } else {
        // ---- results ----
        const int quarter = warp & 3, half = warp >> 2;
        const int tid = threadIdx.x;
        int acc = 0;
        unsigned acc_phase = 0;
        for (int i = blockIdx.x; i < u.units; i += gridDim.x) {
            const ProductUnit t = product_unit(u, i);
            const int row = t.m0 + quarter * 32 + lane;  // of the product
            float2 *col = column + acc * kPN;
            if (kLogits) {
                const int cls = c.cls0 + t.n0 + tid;  // the arrays cover whole tiles
                col[tid] = make_float2(__ldg(c.bias2 + cls), c.cls_scale ? __ldg(c.cls_scale + cls) : 1.0f);
                asm volatile("bar.sync 1, %0;" ::"n"(kPEpilogueWarps * 32) : "memory");
            }
            float scale = 1.4426950408889634f, lse2 = 0.f;
            if (kLogits && c.row_scale) scale *= __ldg(c.row_scale + c.row0 + (row < u.m ? row : 0));
            if (KIND == kLogitGrad && row < u.m) lse2 = __ldg(c.lse2 + row);
            if (!bar_wait(acc_full + acc, acc_phase, gone)) {  // the others may stand at the barrier above: keep coming to it
                if (++acc == kAcc) acc = 0, acc_phase ^= 1;
                continue;
            }
            tc_fence_after();
            const uint32_t d = tmem + acc * kPN + half * 128 + ((uint32_t)quarter << 21);
            const bool there = t.count > 0;  // an empty range of the reduction: zeros
            float v[32];
            if constexpr (KIND == kLogitStats) {
                float mx = -INFINITY, sum = 0.f;
#pragma unroll 1
                for (int j = 0; j < 4; ++j) {
                    tmem_load32(d + 32 * j, v);
                    tmem_load_wait();
                    const float2 *cj = col + half * 128 + 32 * j;
                    float top = mx;
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const float2 b = cj[e];
                        v[e] = __fmaf_rn(v[e] * b.y, scale, b.x);
                        top = fmaxf(top, v[e]);
                    }
                    const float ref = top == -INFINITY ? 0.f : top;
                    sum *= exp2_fast(mx - ref);
#pragma unroll
                    for (int e = 0; e < 32; ++e) sum += exp2_fast(v[e] - ref);
                    mx = top;
                }
                if (row < u.m)
                    c.stats[(int64_t)(t.n0 / 128 + half) * c.row_cap + row] = make_float2(mx, sum);
            } else if constexpr (KIND == kLogitGrad) {
                const int label = row < u.m ? c.label[row] - c.cls0 - t.n0 - half * 128 : -1;
                const bool mine = label >= 0 && label < 128;
                uint16_t *g = c.grad + (int64_t)row * c.grad_ld + t.n0 + half * 128;
                const int64_t plane = (int64_t)c.row_cap * c.grad_ld;
#pragma unroll 1
                for (int j = 0; j < 4; ++j) {
                    tmem_load32(d + 32 * j, v);
                    tmem_load_wait();
                    const float2 *cj = col + half * 128 + 32 * j;
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const float2 b = cj[e];
                        v[e] = row < u.m ? exp2_fast(__fmaf_rn(v[e] * b.y, scale, b.x) - lse2) : 0.f;
                        if (PLANES == 2) v[e] *= kGradScale;
                    }
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        uint4 w;
                        uint32_t *pw = reinterpret_cast<uint32_t *>(&w);
                        if (PLANES == 1) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) pw[e] = pack16<__nv_bfloat16>(v[8 * q + 2 * e], v[8 * q + 2 * e + 1]);
                            *reinterpret_cast<uint4 *>(g + 32 * j + 8 * q) = w;
                        } else {
                            uint4 w1;
                            uint32_t *pw1 = reinterpret_cast<uint32_t *>(&w1);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float x0 = v[8 * q + 2 * e], x1 = v[8 * q + 2 * e + 1];
                                pw[e] = pack16<__half>(x0, x1);
                                const float2 r = __half22float2(*reinterpret_cast<const __half2 *>(pw + e));
                                pw1[e] = pack16<__half>(x0 - r.x, x1 - r.y);
                            }
                            *reinterpret_cast<uint4 *>(g + 32 * j + 8 * q) = w;
                            *reinterpret_cast<uint4 *>(g + plane + 32 * j + 8 * q) = w1;
                        }
                    }
                }
                if (mine) {  // the label's class: the same thread wrote it just now without the -1
                    const float p = (exp2_fast(c.picked2[row] - lse2) - 1.0f) * (PLANES == 2 ? kGradScale : 1.0f);
                    if (PLANES == 1) {
                        reinterpret_cast<__nv_bfloat16 *>(g)[label] = __float2bfloat16_rn(p);
                    } else {
                        const __half p0 = __float2half_rn(p);
                        reinterpret_cast<__half *>(g)[label] = p0;
                        reinterpret_cast<__half *>(g + plane)[label] = __float2half_rn(p - __half2float(p0));
                    }
                }
            } else {
                const bool last = KIND == kWeightGrad && c.gw != nullptr;
                if (KIND == kWeightGrad && t.n0 == 0 && half == 0 && (c.gb != nullptr || c.bias_out != nullptr)) {
                    uint32_t one;
                    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];"
                                 : "=r"(one)
                                 : "r"(tmem + kPN + ((uint32_t)quarter << 21)));
                    tmem_load_wait();
                    const float s = there ? __uint_as_float(one) : 0.f;
                    if (row < u.m) {
                        if (c.bias_out) {
                            float *o = c.bias_out + t.split * c.bias_split + row;
                            *o = c.add ? *o + s : s;
                        } else if (c.gb_f32) {
                            static_cast<float *>(c.gb)[c.cls0 + row] = s * c.scale;
                        } else {
                            static_cast<__nv_bfloat16 *>(c.gb)[c.cls0 + row] = __float2bfloat16_rn(s * c.scale);
                        }
                    }
                }
#pragma unroll 1
                for (int j = 0; j < 4; ++j) {
                    const int k0 = t.n0 + half * 128 + 32 * j;
                    if (k0 >= u.n) break;
                    tmem_load32(d + 32 * j, v);
                    tmem_load_wait();
                    if (!there) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] = 0.f;
                    }
                    if (row < u.m && !last) {  // partial sums: rows of out_ld floats, a multiple of 32
                        float4 *o = reinterpret_cast<float4 *>(c.out + t.split * c.out_split + (int64_t)row * c.out_ld + k0);
#pragma unroll
                        for (int q = 0; q < 8; ++q) {
                            float4 w = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
                            if (c.add) {
                                const float4 old = o[q];
                                w.x += old.x, w.y += old.y, w.z += old.z, w.w += old.w;
                            }
                            o[q] = w;
                        }
                    } else if (row < u.m) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] *= c.scale;
                        if (c.col_scale) {
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (k0 + e < u.n) v[e] *= __ldg(c.col_scale + k0 + e);
                        }
                        const int64_t at = (int64_t)(c.cls0 + row) * c.gw_ld + k0;
                        const bool whole = k0 + 32 <= u.n;
                        if (c.gw_f32) {
                            float *o = static_cast<float *>(c.gw) + at;
                            if (whole && (reinterpret_cast<uintptr_t>(o) & 15) == 0) {
#pragma unroll
                                for (int q = 0; q < 8; ++q)
                                    reinterpret_cast<float4 *>(o)[q] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
                            } else {
#pragma unroll
                                for (int e = 0; e < 32; ++e)
                                    if (k0 + e < u.n) o[e] = v[e];
                            }
                        } else {
                            __nv_bfloat16 *o = static_cast<__nv_bfloat16 *>(c.gw) + at;
                            if (whole && (reinterpret_cast<uintptr_t>(o) & 15) == 0) {
#pragma unroll
                                for (int q = 0; q < 4; ++q) {
                                    uint4 w;
                                    uint32_t *pw = reinterpret_cast<uint32_t *>(&w);
#pragma unroll
                                    for (int e = 0; e < 4; ++e) pw[e] = pack16<__nv_bfloat16>(v[8 * q + 2 * e], v[8 * q + 2 * e + 1]);
                                    reinterpret_cast<uint4 *>(o)[q] = w;
                                }
                            } else {
#pragma unroll
                                for (int e = 0; e < 32; ++e)
                                    if (k0 + e < u.n) o[e] = __float2bfloat16_rn(v[e]);
                            }
                        }
                    }
                    __syncwarp();
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(acc_empty + acc);
            if (++acc == kAcc) acc = 0, acc_phase ^= 1;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (threadIdx.x == 0 && *gone) atomicExch(c.failed, 1);
    if (warp == kPEpilogueWarps + 1) tmem_free(tmem, kPAccCols);
}

}  // namespace sgnn
