// Weight gradient of a linear map whose input was kept as 8-bit codes (sm_100a):
//
//     gW[m, k] = sum_r g[r, m] (zp_r + sc_r code[r, k])  (+ beta gW[m, k])
//              = sum_r (g[r, m] sc_r) code[r, k]  +  sum_r g[r, m] zp_r
//
// The first sum runs on the tensor cores: a code is exact in bf16, and g sc, rounded once, is carried as three bf16 terms, its
// 24 bits, so a tile takes three products where two fp32 operands would take six.  (Two terms, 2^-17 of a value off, took
// 570 us instead of 625 for 600k rows of 512 and 256 columns with the pack, and left the result 2.6e-6 off instead of
// 0.7e-6.)  The second sum does not depend on k: a few fp32 multiply-adds beside the conversion of g.  The activations are
// never restored in memory: one byte an element is read.
//
// A block owns 128 x 256 results and a range of the rows.  Per 32 rows TMA brings 128 columns of g and 256 of the codes
// into shared memory as they are (where an operand is not aligned for it, the threads load it themselves); sixteen warps
// convert them: the terms of g go to tensor memory, a thread for each of its 128 lanes, the codes back to shared memory as the
// swizzled "MN-major" operand that keeps the order of their rows; one thread issues the products.  What bounds the kernel is the
// bandwidth of shared memory (128 bytes a clock: 121 KB a step; 157 KB with the terms of g there as well).
// Tensor memory rounds every addition towards zero, which over thousands of rows would shrink the result by 1e-5 of itself, so
// after 256 rows the sums move on into the fp32 registers of eight other warps.  The partial results of the row ranges are added
// in a fixed order.
#include "row_io.cuh"
#include "umma.cuh"

namespace sgnn {

constexpr int kGM = 128, kGN = 256, kGRows = 32;  // results of a block, rows a step
constexpr int kGKeepers = 8;                      // warps that hold the sums
constexpr int kGWorkers = 16;                     // warps that convert
constexpr int kGOwn = kGRows * 4 / kGWorkers;     // rows of g a converting thread works on at a time
constexpr int kGThreads = (kGKeepers + kGWorkers + 4) * 32;  // and a group of four: one feeds, one issues the products
constexpr int kGRaw = 5, kGStages = 4;            // buffers of operands as they come, and converted
constexpr int kGPromote = 8;                      // steps between two moves into registers
constexpr int kGStageBytes = kGN * kGRows * 2;    // the codes of a step; the terms of g take 48 columns of tensor memory
constexpr int kGTermColumns = 3 * 16;              // of a step: 32 bf16 values a lane and term
constexpr int kGTerms = kGN;                      // where those columns begin, behind the sums

struct GradCall {
    CUtensorMap g, codes, zs;  // zs: params as one long row
    const void *g_ptr;
    int64_t ldg;
    const uint8_t *code_ptr;
    int64_t ldc;
    const float2 *params;
    int64_t n;
    int M, F;
    int tiles_m, tiles_n, steps, per_split;  // steps of kGRows rows, of all and of a split
    float *partials;                         // [splits, M, ld]
    int64_t ld;
    int *failed;
};

// What TMA brings: neither g nor the codes (and parameters), the codes, both; the threads load the rest themselves.  Rows of g
// that follow each other without a gap, whatever their width, come as one run of bytes a step: 32 rows always begin at a
// multiple of 16 bytes (the rows of a last step that is not whole, the threads load).
enum GradFeed { kFeedNone, kFeedCodes, kFeedRows, kFeedBoth };
constexpr int kGRowBytes = 512;  // the longest such row
// Where everything is brought, two groups of eight converting warps take every other step each, twice the work at once: what a
// step waits for (barriers, tensor memory, the fence) then counts half (600k rows of 512 and 256 columns: 620 -> 600 us with the pack).
template <int FEED>
constexpr int kGGroups = FEED >= kFeedRows ? 2 : 1;
template <class T, int FEED>
constexpr int grad_raw_g() { return FEED == kFeedBoth ? kGRows * kGM * (int)sizeof(T) : FEED == kFeedRows ? kGRows * kGRowBytes : 0; }
template <class T, int FEED>
constexpr int grad_raw_bytes() { return FEED == kFeedNone ? 0 : grad_raw_g<T, FEED>() + kGRows * (kGN + 8); }
template <class T, int FEED>
constexpr int grad_raw_area()
{
    const int ring = kGRaw * grad_raw_bytes<T, FEED>(), share = 8 * kGM * 4;  // the shares of the zero points go there last
    return ring > share ? ring : share;
}
template <class T, int FEED>
constexpr int grad_shared_bytes() { return kGStages * kGStageBytes + grad_raw_area<T, FEED>() + 256; }

// Eight codes -> eight bf16 values, exact.  A code c in the low byte below 0x43 reads as 128 + c for c < 128 and as 2 c from
// there on; c is the smaller of that minus 128 and half of it.
__device__ __forceinline__ uint4 code_values(uint2 c)
{
    uint4 out;
    __nv_bfloat162 *o = reinterpret_cast<__nv_bfloat162 *>(&out);
    const uint32_t w[4] = {__byte_perm(c.x, 0x43434343u, 0x4140), __byte_perm(c.x, 0x43434343u, 0x4342),
                           __byte_perm(c.y, 0x43434343u, 0x4140), __byte_perm(c.y, 0x43434343u, 0x4342)};
    const __nv_bfloat162 less = __floats2bfloat162_rn(-128.0f, -128.0f), half = __floats2bfloat162_rn(0.5f, 0.5f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162 *>(w + i);
        o[i] = __hmin2(__hadd2(v, less), __hmul2(v, half));
    }
    return out;
}

__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b)
{
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// two bf16 values, the nearest to x and y, which keep what is left
__device__ __forceinline__ uint32_t next_term(unsigned long long &xy)
{
    float x, y;
    unpk2(xy, x, y);
    const __nv_bfloat162 t = __floats2bfloat162_rn(x, y);
    const uint32_t bits = *reinterpret_cast<const uint32_t *>(&t);
    xy = sub2(xy, pk2(__uint_as_float(bits << 16), __uint_as_float(bits & 0xFFFF0000u)));
    return bits;
}

template <class T, int FEED>
__global__ void __launch_bounds__(kGThreads, 1) weight_grad_kernel(const __grid_constant__ GradCall c)
{
    extern __shared__ __align__(1024) uint8_t base[];
    uint8_t *raw = base + kGStages * kGStageBytes;
    constexpr int kRawBytes = grad_raw_bytes<T, FEED>(), kRawArea = grad_raw_area<T, FEED>();
    constexpr int kGroups = kGGroups<FEED>, kOwnWarps = kGWorkers / kGroups;
    constexpr int kRawG = grad_raw_g<T, FEED>();  // g first, then the codes, then the parameters
    uint64_t *raw_full = reinterpret_cast<uint64_t *>(raw + kRawArea), *raw_empty = raw_full + kGRaw;
    uint64_t *full = raw_empty + kGRaw, *empty = full + kGStages, *acc_full = empty + kGStages, *acc_empty = acc_full + 1;
    uint64_t *drained = acc_empty + 1;
    uint32_t *slot = reinterpret_cast<uint32_t *>(drained + 1);
    volatile int *gone = reinterpret_cast<volatile int *>(slot + 1);
    const int warp = __shfl_sync(FULL, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // the same for a warp, and known to be
    if ((smem_addr(base) & 1023u) != 0) {  // the swizzle counts from 1024-byte boundaries
        if (threadIdx.x == 0) atomicExch(c.failed, 1);
        return;
    }
    const int tile = blockIdx.x % (c.tiles_m * c.tiles_n), split = blockIdx.x / (c.tiles_m * c.tiles_n);
    const int m0 = tile % c.tiles_m * kGM, n0 = tile / c.tiles_m * kGN;
    const int first = split * c.per_split;
    const int count = (first + c.per_split < c.steps ? c.per_split : c.steps - first);  // at least one: see weight_grad_plan
    const int rounds = (count + kGPromote - 1) / kGPromote;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kGRaw; ++s) bar_init(raw_full + s, 1), bar_init(raw_empty + s, kOwnWarps);
        for (int s = 0; s < kGStages; ++s) bar_init(full + s, kOwnWarps), bar_init(empty + s, 1);
        bar_init(acc_full, 1), bar_init(acc_empty, kGKeepers);
        bar_init(drained, 1);
        *gone = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kGKeepers + kGWorkers + 1) tmem_alloc(slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *slot;

    // Registers follow the work: the 28 warps are launched with 72 each, 8 x 152 + 16 x 40 + 4 x 40 = 28 x 72.
    if (warp >= kGKeepers + kGWorkers) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == kGKeepers + kGWorkers) {
            // ---- loads ----
            if (FEED != kFeedNone && lane == 0) {
                if (FEED == kFeedBoth) tma_prefetch(&c.g);
                tma_prefetch(&c.codes);
                tma_prefetch(&c.zs);
                int s = 0, done = 0;
                unsigned phase = 0;
#pragma unroll 1
                for (; done < count; ++done) {
                    if (!bar_wait(raw_empty + s, phase ^ 1, gone)) break;
                    uint8_t *at = raw + s * kRawBytes;
                    const int r0 = (first + done) * kGRows;
                    const unsigned g_bytes = FEED == kFeedRows && r0 + kGRows <= c.n ? kGRows * c.M * (unsigned)sizeof(T) : 0u;
                    bar_expect(raw_full + s, FEED == kFeedRows ? kRawBytes - kRawG + g_bytes : kRawBytes);
                    if (g_bytes) bulk_load(at, static_cast<const T *>(c.g_ptr) + (int64_t)r0 * c.M, g_bytes, raw_full + s);
                    if (FEED == kFeedBoth) tma_load(at, &c.g, m0, r0, 0, raw_full + s);
                    tma_load(at + kRawG, &c.codes, n0, r0, 0, raw_full + s);
                    tma_load(at + kRawG + kGRows * kGN, &c.zs, 2 * r0, 0, 0, raw_full + s);
                    if (++s == kGRaw) s = 0, phase ^= 1;
                }
                if (done < count) ring_drain(raw_full, done, kGRaw);
            }
            __syncwarp();
        } else if (warp == kGKeepers + kGWorkers + 1) {
            // ---- products ----
            if (lane == 0) {
                const int left = c.F - n0, n = left < kGN ? (left + 15) / 16 * 16 : kGN;
                const uint32_t idesc = umma_idesc(true, false, true, n);
                int s = 0;
                unsigned phase = 0;
                bool ok = true;
#pragma unroll 1
                for (int k = 0; k < count; ++k) {
                    if (k % kGPromote == 0) {
                        ok = bar_wait(acc_empty, ((k / kGPromote) & 1) ^ 1, gone);
                        if (!ok) break;
                    }
                    ok = bar_wait(full + s, phase, gone);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t b = umma_desc(base + s * kGStageBytes, kGRows * 128, 1024);
                    const uint32_t a = tmem + kGTerms + s * kGTermColumns;
#pragma unroll
                    for (int j = 0; j < kGRows / 16; ++j) {  // sixteen rows: two groups of eight, eight columns of tensor memory
                        const uint64_t step = 2048u * j >> 4;
                        umma_ts(tmem, a + 8 * j, b + step, idesc, k % kGPromote > 0 || j > 0);
                        umma_ts(tmem, a + 16 + 8 * j, b + step, idesc, true);
                        umma_ts(tmem, a + 32 + 8 * j, b + step, idesc, true);
                    }
                    tc_commit(empty + s);
                    if (k % kGPromote == kGPromote - 1 || k == count - 1) tc_commit(acc_full);
                    if (++s == kGStages) s = 0, phase ^= 1;
                }
                if (!ok) {
                    tc_commit(drained);
                    bar_drain(drained, 0);
                }
            }
            __syncwarp();
        }
    } else if (warp < kGKeepers) {
        // ---- the sums ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 152;");
        const int quarter = warp & 3, half = warp >> 2;  // 32 rows, 128 columns of the results
        float sum[128];
#pragma unroll
        for (int e = 0; e < 128; ++e) sum[e] = 0.f;
#pragma unroll 1
        for (int round = 0; round < rounds; ++round) {
            if (!bar_wait(acc_full, round & 1, gone)) break;
            tc_fence_after();
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float v[16];
                tmem_load16(tmem + half * 128 + 16 * j + ((uint32_t)quarter << 21), v);
                tmem_load_wait(v);
#pragma unroll
                for (int e = 0; e < 16; ++e) sum[16 * j + e] += v[e];
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(acc_empty);
        }
        asm volatile("bar.sync 1, %0;" ::"n"((kGKeepers + kGWorkers) * 32) : "memory");
        const float *share = reinterpret_cast<const float *>(raw);
        const int m = quarter * 32 + lane;
        float own = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) own += share[e * kGM + m] + share[(4 + e) * kGM + m];
        if (m0 + m < c.M) {
            float *o = c.partials + ((int64_t)split * c.M + m0 + m) * c.ld + n0 + half * 128;
#pragma unroll
            for (int e = 0; e < 128; e += 4) {  // ld is F rounded up to 4
                if (n0 + half * 128 + e < c.F)
                    *reinterpret_cast<float4 *>(o + e) = make_float4(sum[e] + own, sum[e + 1] + own, sum[e + 2] + own, sum[e + 3] + own);
            }
        }
    } else {
        // ---- conversion ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        const int w = warp - kGKeepers, group = w / kOwnWarps, own = w % kOwnWarps;
        const int quarter = w & 3, first_row = (own >> 2) * kGOwn * kGroups;  // of g: one column, kGOwn rows, kGroups times
        const int m = quarter * 32 + lane, nq = n0 + lane * 8;  // of the codes: eight columns, rows own, own + kOwnWarps, ...
        const int column = m0 + m < c.M ? m0 + m : 0;  // kFeedRows: lanes beyond the last column work for nothing
        const uint32_t terms = tmem + kGTerms + (first_row >> 1) + ((uint32_t)quarter << 21);
        // sums of g zp: over even and odd steps and over every eight rows of them, whoever has them, for one result whatever FEED is
        float zero[2] = {0.f, 0.f};
        int s = group, t = group;
        unsigned phase = 0, raw_phase = 0;
        // operands of a step that come without TMA, one step ahead
        float gv[kGOwn];
        uint2 cv[kGRows / kOwnWarps];
        const auto fetch = [&](int k) {
            const int64_t r0 = (int64_t)(first + k) * kGRows;
            if constexpr (FEED < kFeedRows) {
#pragma unroll
                for (int i = 0; i < kGOwn; ++i) {
                    const int64_t r = r0 + first_row + i;
                    gv[i] = r < c.n && m0 + m < c.M ? to_f32<T>(static_cast<const T *>(c.g_ptr)[r * c.ldg + m0 + m]) : 0.f;
                }
            }
            if constexpr (FEED == kFeedNone) {
#pragma unroll
                for (int i = 0; i < kGRows / kOwnWarps; ++i) {
                    const int64_t r = r0 + own + kOwnWarps * i;
                    uint8_t b[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) b[e] = r < c.n && nq + e < c.F ? c.code_ptr[r * c.ldc + nq + e] : (uint8_t)0;
                    cv[i].x = b[0] | b[1] << 8 | b[2] << 16 | (uint32_t)b[3] << 24;
                    cv[i].y = b[4] | b[5] << 8 | b[6] << 16 | (uint32_t)b[7] << 24;
                }
            }
        };
        fetch(0);
#pragma unroll 1
        for (int k = group; k < count; k += kGroups) {
            const uint8_t *in = raw + s * kRawBytes;
            if (FEED != kFeedNone && !bar_wait(raw_full + s, raw_phase, gone)) break;
            if (!bar_wait(empty + t, phase ^ 1, gone)) break;
            uint8_t *at = base + t * kGStageBytes;
            const bool whole = (int64_t)(first + k + 1) * kGRows <= c.n;
#pragma unroll
            for (int p = 0; p < kGroups; ++p) {
                float share = 0.f;
                uint32_t term[3][kGOwn / 2];
#pragma unroll
                for (int i = 0; i < kGOwn / 2; ++i) {
                    const int r = first_row + p * kGOwn + 2 * i;
                    float v0, v1;
                    float4 par;  // (zp, sc) of both rows
                    if constexpr (FEED == kFeedBoth) {
                        const T *g = reinterpret_cast<const T *>(in) + r * kGM + m;
                        v0 = to_f32<T>(g[0]), v1 = to_f32<T>(g[kGM]);
                    } else if constexpr (FEED == kFeedRows) {
                        if (whole) {
                            const T *g = reinterpret_cast<const T *>(in) + r * c.M + column;
                            v0 = to_f32<T>(g[0]), v1 = to_f32<T>(g[c.M]);
                        } else {
                            const int64_t row = (int64_t)(first + k) * kGRows + r;
                            const T *g = static_cast<const T *>(c.g_ptr) + row * c.M + column;
                            v0 = row < c.n ? to_f32<T>(g[0]) : 0.f, v1 = row + 1 < c.n ? to_f32<T>(g[c.M]) : 0.f;
                        }
                    } else {
                        v0 = gv[2 * i], v1 = gv[2 * i + 1];
                    }
                    if constexpr (FEED == kFeedNone) {
                        const int64_t row = (int64_t)(first + k) * kGRows + r;
                        const float2 p0 = row < c.n ? __ldg(c.params + row) : make_float2(0.f, 0.f);
                        const float2 p1 = row + 1 < c.n ? __ldg(c.params + row + 1) : make_float2(0.f, 0.f);
                        par = make_float4(p0.x, p0.y, p1.x, p1.y);
                    } else {
                        par = *reinterpret_cast<const float4 *>(in + kRawG + kGRows * kGN + r * 8);
                    }
                    share = __fmaf_rn(v0, par.x, share);
                    share = __fmaf_rn(v1, par.z, share);
                    unsigned long long left = mul2(pk2(v0, v1), pk2(par.y, par.w));
#pragma unroll
                    for (int e = 0; e < 3; ++e) term[e][i] = next_term(left);
                }
#pragma unroll
                for (int e = 0; e < 3; ++e) tmem_store4(terms + t * kGTermColumns + 16 * e + p * (kGOwn / 2), term[e]);
                zero[kGroups == 2 ? p : k & 1] += share;
            }
#pragma unroll
            for (int i = 0; i < kGRows / kOwnWarps; ++i) {
                const int r = own + kOwnWarps * i;
                const uint2 code = FEED == kFeedNone ? cv[i] : *reinterpret_cast<const uint2 *>(in + kRawG + r * kGN + lane * 8);
                *reinterpret_cast<uint4 *>(at + (lane >> 3) * (kGRows * 128) + r * 128 + ((lane & 7) ^ (r & 7)) * 16) = code_values(code);
            }
            tmem_store_wait();
            tc_fence_before();
            if (FEED < kFeedRows && k + kGroups < count) fetch(k + kGroups);
            async_fence();
            __syncwarp();
            if (lane == 0) {
                bar_arrive(full + t);
                if (FEED != kFeedNone) bar_arrive(raw_empty + s);
            }
            if ((t += kGroups) >= kGStages) t -= kGStages, phase ^= 1;
            if ((s += kGroups) >= kGRaw) s -= kGRaw, raw_phase ^= 1;
        }
        // the zero points' shares of every column, [2][4][128]: every buffer of operands as they come has been read by then
        asm volatile("bar.sync 2, %0;" ::"n"(kGWorkers * 32) : "memory");
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const int place = kGroups == 2 ? group * 4 + (own >> 2) * 2 + p : p * 4 + (own >> 2);
            reinterpret_cast<float *>(raw)[place * kGM + m] = zero[p];
        }
        asm volatile("bar.sync 1, %0;" ::"n"((kGKeepers + kGWorkers) * 32) : "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (threadIdx.x == 0 && *gone) atomicExch(c.failed, 1);
    if (warp == kGKeepers + kGWorkers + 1) tmem_free(tmem, 512);
}

// out = sum of the partial results, in their order, + beta out: 32 columns a block row, the splits dealt over eight warps
__global__ void __launch_bounds__(256)
weight_grad_join_kernel(const float *__restrict__ partials, int splits, int M, int F, int64_t ld, float beta,
                        const int *__restrict__ failed, float *__restrict__ out, int64_t ldo)
{
    __shared__ float red[8][33];
    const int lane = threadIdx.x & 31, g = threadIdx.x >> 5;
    const int64_t f = (int64_t)blockIdx.x * 32 + lane;
    const bool bad = splits > 0 && *failed != 0;
    for (int64_t m = blockIdx.y; m < M; m += gridDim.y) {
        float acc = 0.f;
        if (f < F) {
#pragma unroll 4
            for (int s = g; s < splits; s += 8) acc += partials[((int64_t)s * M + m) * ld + f];
        }
        __syncthreads();
        red[g][lane] = acc;
        __syncthreads();
        if (g == 0 && f < F) {
            for (int w = 1; w < 8; ++w) acc += red[w][lane];
            float *o = out + m * ldo + f;
            if (bad) acc = __int_as_float(0x7fffffff);
            *o = beta == 0.f ? acc : acc + beta * *o;
        }
    }
}

struct GradPlan {
    int tiles_m, tiles_n, steps, per_split, splits;
    int64_t ld;
    size_t bytes;
};

// As many row ranges as fill the SMs once, each with at least one move into registers' worth of rows where there are that
// many; every range has rows.
static GradPlan weight_grad_plan(int64_t n, int64_t M, int64_t F)
{
    GradPlan p{};
    p.tiles_m = (int)ceil_div(M, kGM), p.tiles_n = (int)ceil_div(F, kGN);
    p.steps = (int)ceil_div(n, kGRows);
    int64_t s = sm_count() / ((int64_t)p.tiles_m * p.tiles_n);
    const int64_t most = ceil_div(p.steps, kGPromote);
    if (s > most) s = most;
    if (s < 1) s = 1;
    p.per_split = (int)ceil_div(p.steps, s);
    p.splits = (int)ceil_div(p.steps, p.per_split);
    p.ld = ceil_div(F, 4) * 4;
    p.bytes = 256 + (size_t)p.splits * M * p.ld * sizeof(float);
    return p;
}

template <class T, int FEED>
static int weight_grad_launch(const GradCall &c, const GradPlan &p, cudaStream_t s)
{
    constexpr int smem = grad_shared_bytes<T, FEED>();
    static ResidentCache cache;  // one block an SM; asked for the shared memory's attribute
    int resident = 0, rc = resident_blocks(weight_grad_kernel<T, FEED>, kGThreads, smem, smem, cache, &resident);
    if (rc) return rc;
    weight_grad_kernel<T, FEED><<<(unsigned)(p.tiles_m * p.tiles_n * p.splits), kGThreads, smem, s>>>(c);
    SGNN_LAUNCH_OK("checkpoint_weight_grad");
    return SGNN_OK;
}

template <class T>
static int weight_grad_run(const void *g, int64_t ldg, const uint8_t *codes, int64_t ldc, const float2 *params, int64_t n, int M,
                           int F, float beta, float *out, int64_t ldo, void *ws, const GradPlan &p, cudaStream_t s)
{
    GradCall c{};
    c.g_ptr = g, c.ldg = ldg, c.code_ptr = codes, c.ldc = ldc, c.params = params, c.n = n, c.M = M, c.F = F;
    c.tiles_m = p.tiles_m, c.tiles_n = p.tiles_n, c.steps = p.steps, c.per_split = p.per_split, c.ld = p.ld;
    c.failed = static_cast<int *>(ws), c.partials = reinterpret_cast<float *>(static_cast<char *>(ws) + 256);
    SGNN_CUDA_OK(cudaMemsetAsync(c.failed, 0, 4, s));
    int rc;
    const bool codes_fed = n > 1 && n <= (1ll << 29) && aligned16(codes) && ldc % 16 == 0 && aligned16(params);
    const bool g_fed = codes_fed && aligned16(g) && ldg * sizeof(T) % 16 == 0;
    if (codes_fed) {
        if ((rc = raw_tensor_map(&c.zs, params, 4, 2 * n, 1, ceil_div(n, 2) * 4, 2 * kGRows, 1))) return rc;
        if ((rc = raw_tensor_map(&c.codes, codes, 1, F, n, ldc, kGN, kGRows))) return rc;
    }
    if (g_fed) {
        if ((rc = raw_tensor_map(&c.g, g, sizeof(T), M, n, ldg, kGM, kGRows))) return rc;
        rc = weight_grad_launch<T, kFeedBoth>(c, p, s);
    } else if (codes_fed && aligned16(g) && ldg == M && M * (int)sizeof(T) <= kGRowBytes) {
        rc = weight_grad_launch<T, kFeedRows>(c, p, s);
    } else if (codes_fed) {
        rc = weight_grad_launch<T, kFeedCodes>(c, p, s);
    } else {
        rc = weight_grad_launch<T, kFeedNone>(c, p, s);
    }
    if (rc) return rc;
    const dim3 grid((unsigned)ceil_div(F, 32), (unsigned)(M < 65535 ? M : 65535));
    weight_grad_join_kernel<<<grid, 256, 0, s>>>(c.partials, p.splits, M, F, p.ld, beta, c.failed, out, ldo);
    SGNN_LAUNCH_OK("checkpoint_weight_grad join");
    return SGNN_OK;
}

static int weight_grad_check(const char *who, int dtype, int64_t n, int64_t M, int64_t F)
{
    SGNN_REQUIRE(elem_known(dtype), SGNN_ERR_INVALID_ARGUMENT, "%s: unknown element type", who);
    SGNN_REQUIRE(n >= 0 && M > 0 && F > 0, SGNN_ERR_INVALID_ARGUMENT, "%s: bad size", who);
    SGNN_REQUIRE(n < (1LL << 31) && M <= 65536 && F <= 65536, SGNN_ERR_TOO_LARGE, "%s: too large", who);
    return SGNN_OK;
}

}  // namespace sgnn

using namespace sgnn;

extern "C" SGNN_API int sgnn_checkpoint_weight_grad_workspace_bytes(int dtype, int64_t n, int64_t M, int64_t F, size_t *bytes)
{
    const char *who = "checkpoint_weight_grad_workspace_bytes";
    int rc = weight_grad_check(who, dtype, n, M, F);
    if (rc) return rc;
    SGNN_REQUIRE(bytes != nullptr, SGNN_ERR_INVALID_ARGUMENT, "%s: null result pointer", who);
    *bytes = n == 0 ? 0 : weight_grad_plan(n, M, F).bytes;
    return SGNN_OK;
}

extern "C" SGNN_API int sgnn_checkpoint_weight_grad(int dtype, const void *d_g, int64_t ldg, const uint8_t *d_codes,
                                                    int64_t ldc, const float *d_params, int64_t n, int64_t M, int64_t F,
                                                    float beta, float *d_out, int64_t ldo, void *d_workspace,
                                                    size_t workspace_bytes, void *stream)
{
    const char *who = "checkpoint_weight_grad";
    int rc = weight_grad_check(who, dtype, n, M, F);
    if (rc) return rc;
    SGNN_REQUIRE(beta == beta, SGNN_ERR_INVALID_ARGUMENT, "%s: beta is NaN", who);
    SGNN_REQUIRE(d_out != nullptr && ldo >= F && reinterpret_cast<uintptr_t>(d_out) % 4 == 0, SGNN_ERR_INVALID_ARGUMENT,
                 "%s: bad output", who);
    cudaStream_t s = (cudaStream_t)stream;
    if (n == 0) {
        const dim3 grid((unsigned)ceil_div(F, 32), (unsigned)(M < 65535 ? M : 65535));
        weight_grad_join_kernel<<<grid, 256, 0, s>>>(nullptr, 0, (int)M, (int)F, F, beta, nullptr, d_out, ldo);
        SGNN_LAUNCH_OK("checkpoint_weight_grad join");
        return SGNN_OK;
    }
    SGNN_REQUIRE(d_g && d_codes && d_params, SGNN_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
    SGNN_REQUIRE(n == 1 || (ldg >= M && ldc >= F), SGNN_ERR_INVALID_ARGUMENT, "%s: leading dimension shorter than a row", who);
    SGNN_REQUIRE(reinterpret_cast<uintptr_t>(d_g) % elem_bytes(dtype) == 0 && reinterpret_cast<uintptr_t>(d_params) % 8 == 0,
                 SGNN_ERR_INVALID_ARGUMENT, "%s: pointers must be aligned to their element (params: 8 bytes)", who);
    const GradPlan p = weight_grad_plan(n, M, F);
    SGNN_REQUIRE(d_workspace != nullptr && workspace_bytes >= p.bytes && reinterpret_cast<uintptr_t>(d_workspace) % 256 == 0,
                 SGNN_ERR_WORKSPACE, "%s: 256-byte aligned workspace of %zu bytes needed, %zu given", who, p.bytes, workspace_bytes);
    const float2 *params = reinterpret_cast<const float2 *>(d_params);
    const int m = (int)M, f = (int)F;
    if (dtype == SGNN_F32) return weight_grad_run<float>(d_g, ldg, d_codes, ldc, params, n, m, f, beta, d_out, ldo, d_workspace, p, s);
    if (dtype == SGNN_BF16) return weight_grad_run<__nv_bfloat16>(d_g, ldg, d_codes, ldc, params, n, m, f, beta, d_out, ldo, d_workspace, p, s);
    return weight_grad_run<__half>(d_g, ldg, d_codes, ldc, params, n, m, f, beta, d_out, ldo, d_workspace, p, s);
}
