// Layer norm of the rows of a matrix and its gradients (sm_100a):
//
//     mean = sum_c x[c] / H,  rstd = 1 / sqrt(sum_c (x[c] - mean)^2 / H + eps),  xh = (x - mean) rstd
//     y  = xh gamma + beta
//     gx = rstd (a - mean(a) - xh mean(a xh)),  a = gy gamma
//     grad_gamma[c] = sum_r gy[r, c] xh[r, c],  grad_beta[c] = sum_r gy[r, c]
//
// The reference calls torch.nn.LayerNorm between two layers (examples/graphsage/sage.py:149-151, 192-194).  The
// forward can write the 8-bit checkpoint of x in the same pass, and the backward can read that checkpoint in place of
// x: one byte an element kept between the two instead of four.
//
// Everything is bound by memory: the forward moves x and y once, the backward gy, x (or its codes) and gx once.  Rows
// belong to a warp, narrow ones to 4, 8 or 16 of its lanes, which hold them in registers between the reductions and the
// outputs: forward up to 2048 elements where accesses of 16 bytes or the ring of bulk copies apply and 1024 elsewhere;
// backward up to 832 (kNormSplit), 16-bit rows through the ring up to 1024, from codes up to 512 unless fp32 rows lie on
// boundaries.  Backward up to 2048 they belong to a block that does the same; longer rows to a block that reads them again
// (from L1 / L2) for every step: 30000 x 4096 fp32 220 us forward of 150 that the bytes take, 528 of 226 backward.  All sums
// are fp32: the variance from the differences to the mean, the column sums per warp, then per block, then over the blocks,
// in a fixed order.
#include "row_io.cuh"
#include "umma.cuh"

namespace sgnn {

constexpr int kNormThreads = 256;
constexpr int kNormWarps = kNormThreads / 32;
constexpr int kNormMaxWidth = 16384;  // the block kernels keep two column sums an element in shared memory

struct NormParam {
    const void *gamma, *beta;  // nullptr: 1 and 0
    bool f32;                  // fp32, otherwise of the activation type
};

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------
// CK: also write the 8-bit codes of x and their (zero point, scale)
template <class T, int E, int NV, bool CK, int LANES>
__global__ void __launch_bounds__(kNormThreads)
norm_fwd_warp_kernel(const T *__restrict__ x, int64_t ldx, NormParam par, float eps, T *__restrict__ y, int64_t ldy,
                     float2 *__restrict__ stats, uint8_t *__restrict__ codes, int64_t ldc, float2 *__restrict__ params,
                     int64_t n, int H)
{
    constexpr bool kHold = E * NV <= 8;  // gamma and beta in registers; from L1 every row where they would not fit
    constexpr int kRows = 32 / LANES;  // of a warp at a time
    const int lane = threadIdx.x % LANES, sub = (threadIdx.x & 31) / LANES;
    const float invH = 1.0f / (float)H;
    float ga[kHold ? NV : 1][E], be[kHold ? NV : 1][E];
    if constexpr (kHold) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (lane + LANES * i) * E;
            if (c < H) {
                load_param<T, E>(par.gamma, par.f32, c, 1.f, ga[i]);
                load_param<T, E>(par.beta, par.f32, c, 0.f, be[i]);
            }
        }
    }
    const int64_t step = (int64_t)gridDim.x * kNormWarps * kRows;
    for (int64_t r0 = ((int64_t)blockIdx.x * kNormWarps + (threadIdx.x >> 5)) * kRows; r0 < n; r0 += step) {
        const int64_t r = r0 + sub;
        const int width = r < n ? H : 0;
        float v[NV][E];
        float s = 0.f, mn = INFINITY, mx = -INFINITY, poison = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (lane + LANES * i) * E;
            if (c < width) load_row<T, E>(x + r * ldx + c, v[i]);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if ((lane + LANES * i) * E < width) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    s += v[i][e];
                    if (CK) {
                        mn = fminf(mn, v[i][e]);
                        mx = fmaxf(mx, v[i][e]);
                        poison = __fmaf_rn(v[i][e], 0.f, poison);
                    }
                }
            }
        }
        const float mean = row_sum<LANES>(s) * invH;
        float q = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if ((lane + LANES * i) * E < width) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float d = v[i][e] - mean;
                    q += d * d;
                }
            }
        }
        const float rstd = __frsqrt_rn(row_sum<LANES>(q) * invH + eps);
        if (lane == 0 && r < n) stats[r] = make_float2(mean, rstd);
        RowQ rq;
        if (CK) {
            rq = row_quantiser(row_min<LANES>(mn), row_max<LANES>(mx), row_sum<LANES>(poison));
            if (lane == 0 && r < n) params[r] = make_float2(rq.mn, rq.sc);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (lane + LANES * i) * E;
            if (c < width) {
                if (CK) store_codes<E>(codes + r * ldc + c, v[i], rq);
                float g[E], b[E];
                if constexpr (!kHold) {
                    load_param<T, E>(par.gamma, par.f32, c, 1.f, g);
                    load_param<T, E>(par.beta, par.f32, c, 0.f, b);
                }
                float o[E];
#pragma unroll
                for (int e = 0; e < E; ++e)
                    o[e] = (v[i][e] - mean) * rstd * (kHold ? ga[kHold ? i : 0][e] : g[e]) + (kHold ? be[kHold ? i : 0][e] : b[e]);
                store_row<T, E>(y + r * ldy + c, o);
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Packed rows that do not start on 16-byte boundaries (602 bf16 columns, say).  Eight rows together do: they are one run of
// memory of a multiple of 16 bytes, which a bulk copy brings into shared memory whatever the width.  A block walks over
// batches of eight rows, a row a warp, through a ring of such buffers: the copies of the next batches run while one is
// computed, and the results go back from the buffer they were computed in.  With loads of one or two elements a thread instead,
// 100003 x 602 in bf16 took 117 us forward and 303 us backward (too few bytes on their way, and 146 registers).
// ---------------------------------------------------------------------------
constexpr int kStagedMax = 4;             // buffers of the ring
constexpr size_t kStagedCap = 160 * 1024;  // shared memory of a block
constexpr int kStagedForward = 2048;       // longest rows of the forward; of the backward 1024 of 16 bits, kNormSplit of fp32
// two buffers of eight such fp32 rows and gamma and beta (147 KB), two of two operands and gamma (110 KB)
static_assert(2 * kNormWarps * kStagedForward * 4 + 2 * kStagedForward * 4 <= kStagedCap);

struct StagedRing {
    uint8_t *base;  // buffer s at base + s * stride; the second operand of the backward `second` bytes behind
    size_t stride, second;
    int depth;
};

// 8 H sizeof(T) bytes from each of one or two operands into buffer s, one fill more; the last batch of a matrix may be short and is
// copied by the threads.
template <class T>
__device__ __forceinline__ void staged_load(const StagedRing &ring, int s, const T *p, const T *q, int64_t batch, int64_t full, int64_t n,
                                            int H, uint64_t *bar, unsigned &used)
{
    if (batch >= full || threadIdx.x != 0) return;
    ++used;
    const unsigned bytes = (unsigned)(kNormWarps * H * sizeof(T));
    uint8_t *at = ring.base + s * ring.stride;
    bar_expect(bar, q ? 2 * bytes : bytes);
    bulk_load(at, p + batch * kNormWarps * H, bytes, bar);
    if (q) bulk_load(at + ring.second, q + batch * kNormWarps * H, bytes, bar);
}
template <class T>
__device__ __forceinline__ void staged_copy_in(T *dst, const T *src, int64_t batch, int64_t n, int H)
{
    const int64_t first = batch * kNormWarps * H, count = n * H - first;
    for (int64_t i = threadIdx.x; i < count; i += kNormThreads) dst[i] = src[first + i];
}
template <class T>
__device__ __forceinline__ void staged_copy_out(T *dst, const T *src, int64_t batch, int64_t n, int H)
{
    const int64_t first = batch * kNormWarps * H, count = n * H - first;
    for (int64_t i = threadIdx.x; i < count; i += kNormThreads) dst[first + i] = src[i];
}

template <class T, int E>
__device__ __forceinline__ void shared_get(const T *p, float (&v)[E])
{
    union {
        typename Word<E * sizeof(T)>::type w;
        T e[E];
    } u;
    u.w = *reinterpret_cast<const typename Word<E * sizeof(T)>::type *>(p);
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = to_f32<T>(u.e[i]);
}
template <class T, int E>
__device__ __forceinline__ void shared_put(T *p, const float (&v)[E])
{
    union {
        typename Word<E * sizeof(T)>::type w;
        T e[E];
    } u;
#pragma unroll
    for (int i = 0; i < E; ++i) u.e[i] = from_f32<T>(v[i]);
    *reinterpret_cast<typename Word<E * sizeof(T)>::type *>(p) = u.w;
}

// One walk over the batches of a block: `row(data, other, r)` computes a row of this warp in place of `data`.
// Every wait is for a copy this block has issued.  *gone: a copy did not come within the bound; no result is written from then
// on, and a NaN in the statistics or the column sums says so.
template <class T, class Row>
__device__ __forceinline__ void staged_walk(const StagedRing &ring, const T *p, const T *q, T *out, int64_t n, int H, uint64_t *full_bar,
                                            volatile int *gone, Row row)
{
    const int64_t batches = (n + kNormWarps - 1) / kNormWarps, full = n / kNormWarps;
    const int warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        for (int s = 0; s < ring.depth; ++s) bar_init(full_bar + s, 1);
        *gone = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    unsigned used = 0;  // fills by thread 0: buffer 0, 1, ..., 0, 1, ...
    for (int s = 0; s < ring.depth; ++s)
        if ((int64_t)blockIdx.x + (int64_t)s * gridDim.x < batches)
            staged_load(ring, s, p, q, (int64_t)blockIdx.x + (int64_t)s * gridDim.x, full, n, H, full_bar + s, used);
    int s = 0;
    unsigned phase = 0;
    for (int64_t b = blockIdx.x; b < batches; b += gridDim.x) {
        T *data = reinterpret_cast<T *>(ring.base + s * ring.stride);
        T *other = reinterpret_cast<T *>(ring.base + s * ring.stride + ring.second);
        if (b < full) {
            bar_wait(full_bar + s, phase, gone);
        } else {
            // ordinary stores by every thread into a buffer whose result of an earlier batch left it by a bulk store of thread 0's:
            // it has to have been read (with two buffers no barrier since thread 0's last wait says so)
            if (threadIdx.x == 0) store_wait_read();
            __syncthreads();
            staged_copy_in(data, p, b, n, H);
            if (q) staged_copy_in(other, q, b, n, H);
            __syncthreads();
        }
        const int64_t r = b * kNormWarps + warp;
        if (r < n) row(data + (size_t)warp * H, other + (size_t)warp * H, r);
        async_fence();
        __syncthreads();
        if (*gone) break;  // the same for every thread: read after the barrier, written before it
        if (b >= full) {
            staged_copy_out(out, data, b, n, H);  // the last batch of all
        } else if (threadIdx.x == 0) {
            bulk_store(out + b * kNormWarps * H, data, (unsigned)(kNormWarps * H * sizeof(T)));
            store_commit();
        }
        // refill the buffer before this one: its store was issued a batch ago
        const int64_t next = b + (int64_t)(ring.depth - 1) * gridDim.x;
        if (b != blockIdx.x && next < batches) {
            const int before = s == 0 ? ring.depth - 1 : s - 1;
            if (threadIdx.x == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
            staged_load(ring, before, p, q, next, full, n, H, full_bar + before, used);
        }
        if (++s == ring.depth) s = 0, phase ^= 1;
    }
    if (threadIdx.x == 0) {
        store_wait_all();
        if (*gone) ring_drain(full_bar, used, ring.depth);
    }
}

template <class T, int E, int NV>
__global__ void __launch_bounds__(kNormThreads)
norm_fwd_staged_kernel(const T *__restrict__ x, NormParam par, float eps, T *__restrict__ y, float2 *__restrict__ stats, int64_t n, int H,
                       size_t stride, int depth)
{
    extern __shared__ __align__(128) uint8_t area[];
    __shared__ uint64_t bars[kStagedMax];
    __shared__ int gone;
    float *ga = reinterpret_cast<float *>(area), *be = ga + H;
    for (int c = threadIdx.x; c < H; c += kNormThreads) {
        float g[1], b[1];
        load_param<T, 1>(par.gamma, par.f32, c, 1.f, g);
        load_param<T, 1>(par.beta, par.f32, c, 0.f, b);
        ga[c] = g[0], be[c] = b[0];
    }
    const StagedRing ring{area + ((size_t)2 * H * sizeof(float) + 127) / 128 * 128, stride, 0, depth};
    const int lane = threadIdx.x & 31;
    const float invH = 1.0f / (float)H;
    staged_walk<T>(ring, x, static_cast<const T *>(nullptr), y, n, H, bars, &gone, [&](T *data, T *, int64_t r) {
        float v[NV][E];
        float s = 0.f, q = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (lane + 32 * i) * E;
            if (c < H) {
                shared_get<T, E>(data + c, v[i]);
#pragma unroll
                for (int e = 0; e < E; ++e) s += v[i][e];
            }
        }
        const float mean = all_sum(s) * invH;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if ((lane + 32 * i) * E < H) {
#pragma unroll
                for (int e = 0; e < E; ++e) v[i][e] -= mean, q += v[i][e] * v[i][e];
            }
        }
        const float rstd = __frsqrt_rn(all_sum(q) * invH + eps);
        if (lane == 0) stats[r] = make_float2(mean, rstd);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (lane + 32 * i) * E;
            if (c < H) {
#pragma unroll
                for (int e = 0; e < E; ++e) v[i][e] = v[i][e] * rstd * ga[c + e] + be[c + e];
                shared_put<T, E>(data + c, v[i]);
            }
        }
    });
    if (threadIdx.x == 0 && gone) stats[blockIdx.x % n] = make_float2(__int_as_float(0x7fffffff), __int_as_float(0x7fffffff));
}

template <class T, int E, int NV>
__global__ void __launch_bounds__(kNormThreads)
norm_bwd_staged_kernel(const T *__restrict__ gy, const T *__restrict__ x, const float2 *__restrict__ stats, NormParam par,
                       T *__restrict__ gx, float *__restrict__ partials, int64_t n, int H, size_t stride, size_t second, int depth)
{
    extern __shared__ __align__(128) uint8_t area[];
    __shared__ uint64_t bars[kStagedMax];
    __shared__ int gone;
    float *ga = reinterpret_cast<float *>(area);
    for (int c = threadIdx.x; c < H; c += kNormThreads) {
        float g[1];
        load_param<T, 1>(par.gamma, par.f32, c, 1.f, g);
        ga[c] = g[0];
    }
    const StagedRing ring{area + ((size_t)H * sizeof(float) + 127) / 128 * 128, stride, second, depth};
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float invH = 1.0f / (float)H;
    float sg[NV][E], sb[NV][E];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) sg[i][e] = sb[i][e] = 0.f;
    staged_walk<T>(ring, gy, x, gx, n, H, bars, &gone, [&](T *data, T *other, int64_t r) {
        float a[NV][E], xh[NV][E];
        const float2 st = __ldg(stats + r);
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (lane + 32 * i) * E;
            if (c < H) {
                shared_get<T, E>(data + c, a[i]);
                shared_get<T, E>(other + c, xh[i]);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    xh[i][e] = (xh[i][e] - st.x) * st.y;
                    sg[i][e] += a[i][e] * xh[i][e];
                    sb[i][e] += a[i][e];
                    a[i][e] *= ga[c + e];
                    s1 += a[i][e];
                    s2 += a[i][e] * xh[i][e];
                }
            }
        }
        const float m1 = all_sum(s1) * invH, m2 = all_sum(s2) * invH;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (lane + 32 * i) * E;
            if (c < H) {
#pragma unroll
                for (int e = 0; e < E; ++e) a[i][e] = st.y * (a[i][e] - m1 - xh[i][e] * m2);
                shared_put<T, E>(data + c, a[i]);
            }
        }
    });
    __syncthreads();
    // the block's column sums: the buffers are free (the last store from them has been waited for)
    float *sums = reinterpret_cast<float *>(ring.base);
    const float bad = gone ? __int_as_float(0x7fffffff) : 0.f;
    for (int w = 0; w < kNormWarps; ++w) {  // one warp after the other
        if (warp == w) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (lane + 32 * i) * E;
                if (c < H) {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        sums[c + e] = (w ? sums[c + e] : bad) + sg[i][e];
                        sums[H + c + e] = (w ? sums[H + c + e] : bad) + sb[i][e];
                    }
                }
            }
        }
        __syncthreads();
    }
    for (int k = threadIdx.x; k < 2 * H; k += kNormThreads) partials[(size_t)blockIdx.x * 2 * H + k] = sums[k];
}

// sum over the block, the same value in every thread
__device__ __forceinline__ float block_sum(float v, float *red)
{
    v = all_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < kNormWarps; ++w) t += red[w];
    return t;
}

__device__ __forceinline__ float block_max(float v, float *red)
{
    v = redux_max(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = -INFINITY;
#pragma unroll
    for (int w = 0; w < kNormWarps; ++w) t = fmaxf(t, red[w]);
    return t;
}

template <class T, int E, bool CK>
__global__ void __launch_bounds__(kNormThreads)
norm_fwd_block_kernel(const T *__restrict__ x, int64_t ldx, NormParam par, float eps, T *__restrict__ y, int64_t ldy,
                      float2 *__restrict__ stats, uint8_t *__restrict__ codes, int64_t ldc,
                      float2 *__restrict__ params, int64_t n, int H)
{
    __shared__ float red[kNormWarps];
    const float invH = 1.0f / (float)H;
    for (int64_t r = blockIdx.x; r < n; r += gridDim.x) {
        const T *xr = x + r * ldx;
        float s = 0.f, mn = INFINITY, mx = -INFINITY, poison = 0.f, v[E];
        for (int c = threadIdx.x * E; c < H; c += kNormThreads * E) {
            load_row<T, E>(xr + c, v);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                s += v[e];
                if (CK) mn = fminf(mn, v[e]), mx = fmaxf(mx, v[e]), poison = __fmaf_rn(v[e], 0.f, poison);
            }
        }
        const float mean = block_sum(s, red) * invH;
        float q = 0.f;
        for (int c = threadIdx.x * E; c < H; c += kNormThreads * E) {
            load_row<T, E>(xr + c, v);
#pragma unroll
            for (int e = 0; e < E; ++e) q += (v[e] - mean) * (v[e] - mean);
        }
        const float rstd = __frsqrt_rn(block_sum(q, red) * invH + eps);
        RowQ rq;
        if (CK) rq = row_quantiser(-block_max(-mn, red), block_max(mx, red), block_sum(poison, red));
        if (threadIdx.x == 0) {
            stats[r] = make_float2(mean, rstd);
            if (CK) params[r] = make_float2(rq.mn, rq.sc);
        }
        for (int c = threadIdx.x * E; c < H; c += kNormThreads * E) {
            float g[E], b[E];
            load_row<T, E>(xr + c, v);
            load_param<T, E>(par.gamma, par.f32, c, 1.f, g);
            load_param<T, E>(par.beta, par.f32, c, 0.f, b);
            if (CK) store_codes<E>(codes + r * ldc + c, v, rq);
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = (v[e] - mean) * rstd * g[e] + b[e];
            store_row<T, E>(y + r * ldy + c, v);
        }
    }
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------
// Where the backward finds xh: x itself, or the 8-bit codes of x (then xh = code (sc rstd) + (zp - mean) rstd)
struct NormSource {
    const void *x;
    int64_t ldx;
    const uint8_t *codes;
    int64_t ldc;
    const float2 *params;
};

struct NormAffine {
    float mul, add;  // xh = value * mul + add, value = x or its code
};

template <bool CK>
__device__ __forceinline__ NormAffine norm_affine(const NormSource &src, int64_t r, float2 st)
{
    NormAffine f;
    if (CK) {
        const float2 p = __ldg(src.params + r);
        f.mul = p.y * st.y;
        f.add = (p.x - st.x) * st.y;
    } else {
        f.mul = st.y;
        f.add = -st.x;  // (x + add) * mul
    }
    return f;
}

template <bool CK>
__device__ __forceinline__ float norm_hat(float v, NormAffine f)
{
    return CK ? __fmaf_rn(v, f.mul, f.add) : (v + f.add) * f.mul;
}

template <class T, int E, bool CK>
__device__ __forceinline__ void load_source(const NormSource &src, int64_t r, int c, float (&v)[E])
{
    if constexpr (CK) load_codes<E>(src.codes + r * src.ldc + c, v);
    else load_row<T, E>(static_cast<const T *>(src.x) + r * src.ldx + c, v);
}

// partials: [gridDim.x, 2, H], per-block column sums of (gy xh, gy).  From codes, with a byte an element instead of four to wait
// for, a fourth block an SM is worth more than registers (600000 x 256 fp32: 270 us against 295; from x 283 against 277).
template <class T, int E, int NV, bool CK, int LANES>
__global__ void __launch_bounds__(kNormThreads, CK && E * NV <= 8 ? 4 : 1)
norm_bwd_warp_kernel(const T *__restrict__ gy, int64_t ldg, NormSource src, const float2 *__restrict__ stats,
                     NormParam par, T *__restrict__ gx, int64_t ldgx, float *__restrict__ partials, int64_t n, int H)
{
    extern __shared__ float sums[];  // [warps, 2, H]: every lane touches its own columns only until the last step
    constexpr bool kHold = E * NV <= 8;  // the column sums of longer rows live in shared memory
    constexpr int kRows = 32 / LANES;  // of a warp at a time
    const int lane = threadIdx.x % LANES, sub = (threadIdx.x & 31) / LANES, warp = threadIdx.x >> 5;
    float *mine = sums + (size_t)warp * 2 * H;
    const float invH = 1.0f / (float)H;
    float ga[kHold ? NV : 1][E], sg[kHold ? NV : 1][E], sb[kHold ? NV : 1][E];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (lane + LANES * i) * E;
        if constexpr (kHold) {
            if (c < H) load_param<T, E>(par.gamma, par.f32, c, 1.f, ga[i]);
#pragma unroll
            for (int e = 0; e < E; ++e) sg[i][e] = sb[i][e] = 0.f;
        } else if (c < H) {
#pragma unroll
            for (int e = 0; e < E; ++e) mine[c + e] = mine[H + c + e] = 0.f;
        }
    }
    const int64_t step = (int64_t)gridDim.x * kNormWarps * kRows;
    for (int64_t r0 = ((int64_t)blockIdx.x * kNormWarps + warp) * kRows; r0 < n; r0 += step) {
        const int64_t r = r0 + sub;
        const int width = r < n ? H : 0;
        float a[NV][E], xh[NV][E];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (lane + LANES * i) * E;
            if (c < width) {
                load_row<T, E>(gy + r * ldg + c, a[i]);
                load_source<T, E, CK>(src, r, c, xh[i]);
            }
        }
        const int64_t known = r < n ? r : 0;
        const float2 st = __ldg(stats + known);
        const NormAffine f = norm_affine<CK>(src, known, st);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (lane + LANES * i) * E;
            if (c < width) {
                float g[E];
                if constexpr (!kHold) load_param<T, E>(par.gamma, par.f32, c, 1.f, g);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    xh[i][e] = norm_hat<CK>(xh[i][e], f);
                    if constexpr (kHold) {
                        sg[i][e] += a[i][e] * xh[i][e];
                        sb[i][e] += a[i][e];
                    } else {
                        mine[c + e] += a[i][e] * xh[i][e];
                        mine[H + c + e] += a[i][e];
                    }
                    a[i][e] *= kHold ? ga[kHold ? i : 0][e] : g[e];
                    s1 += a[i][e];
                    s2 += a[i][e] * xh[i][e];
                }
            }
        }
        const float m1 = row_sum<LANES>(s1) * invH, m2 = row_sum<LANES>(s2) * invH;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (lane + LANES * i) * E;
            if (c < width) {
#pragma unroll
                for (int e = 0; e < E; ++e) a[i][e] = st.y * (a[i][e] - m1 - xh[i][e] * m2);
                store_row<T, E>(gx + r * ldgx + c, a[i]);
            }
        }
    }
    if constexpr (kHold) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {  // the rows of a warp together
#pragma unroll
            for (int e = 0; e < E; ++e) {
#pragma unroll
                for (int o = 16; o >= LANES; o >>= 1) {
                    sg[i][e] += __shfl_xor_sync(FULL, sg[i][e], o);
                    sb[i][e] += __shfl_xor_sync(FULL, sb[i][e], o);
                }
            }
            const int c = (lane + LANES * i) * E;
            if (c < H) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if (sub == 0) mine[c + e] = sg[i][e], mine[H + c + e] = sb[i][e];
                }
            }
        }
    }
    __syncthreads();
    for (int k = threadIdx.x; k < 2 * H; k += kNormThreads) {
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < kNormWarps; ++w) t += sums[(size_t)w * 2 * H + k];
        partials[(size_t)blockIdx.x * 2 * H + k] = t;
    }
}

// Rows of up to 2048 elements by a block: eight columns a thread, whose sums stay in registers; the row is read once, with one
// barrier.  For rows of more than kNormSplit elements, and from codes, unless fp32 rows lie on boundaries, of more than 512
// (both directions, 100000 rows: 1023 fp32 449 us, 553 through the ring; 1024 fp32 422, 452 by a warp; 800 fp32 379, 370; from
// codes 1024 bf16 403, 605 by a warp; 576 bf16 365, 433; 640 fp32 347, 296).
constexpr int kNormWide = 8 * kNormThreads, kNormSplit = 832;
static_assert(2 * 2 * kNormWarps * kNormSplit * 4 + kNormSplit * 4 <= kStagedCap && 2 * 2 * kNormWarps * 1024 * 2 + 1024 * 4 <= kStagedCap);
template <class T, int E, bool CK>
__global__ void __launch_bounds__(kNormThreads, 3)
norm_bwd_wide_kernel(const T *__restrict__ gy, int64_t ldg, NormSource src, const float2 *__restrict__ stats,
                     NormParam par, T *__restrict__ gx, int64_t ldgx, float *__restrict__ partials, int64_t n, int H)
{
    constexpr int NV = 8 / E;
    __shared__ float2 red[2][kNormWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float invH = 1.0f / (float)H;
    float ga[NV][E], sg[NV][E], sb[NV][E];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (threadIdx.x + kNormThreads * i) * E;
        if (c < H) load_param<T, E>(par.gamma, par.f32, c, 1.f, ga[i]);
#pragma unroll
        for (int e = 0; e < E; ++e) sg[i][e] = sb[i][e] = 0.f;
    }
    int turn = 0;
    for (int64_t r = blockIdx.x; r < n; r += gridDim.x, turn ^= 1) {
        float a[NV][E], xh[NV][E];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (threadIdx.x + kNormThreads * i) * E;
            if (c < H) {
                load_row<T, E>(gy + r * ldg + c, a[i]);
                load_source<T, E, CK>(src, r, c, xh[i]);
            }
        }
        const float2 st = __ldg(stats + r);
        const NormAffine f = norm_affine<CK>(src, r, st);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if ((threadIdx.x + kNormThreads * i) * E < H) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    xh[i][e] = norm_hat<CK>(xh[i][e], f);
                    sg[i][e] += a[i][e] * xh[i][e];
                    sb[i][e] += a[i][e];
                    a[i][e] *= ga[i][e];
                    s1 += a[i][e];
                    s2 += a[i][e] * xh[i][e];
                }
            }
        }
        s1 = all_sum(s1), s2 = all_sum(s2);
        if (lane == 0) red[turn][warp] = make_float2(s1, s2);
        __syncthreads();  // whoever comes back to this half of red has passed the next row's barrier
        float m1 = 0.f, m2 = 0.f;
#pragma unroll
        for (int w = 0; w < kNormWarps; ++w) m1 += red[turn][w].x, m2 += red[turn][w].y;
        m1 *= invH, m2 *= invH;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (threadIdx.x + kNormThreads * i) * E;
            if (c < H) {
#pragma unroll
                for (int e = 0; e < E; ++e) a[i][e] = st.y * (a[i][e] - m1 - xh[i][e] * m2);
                store_row<T, E>(gx + r * ldgx + c, a[i]);
            }
        }
    }
    float *out = partials + (size_t)blockIdx.x * 2 * H;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (threadIdx.x + kNormThreads * i) * E;
        if (c < H) {
#pragma unroll
            for (int e = 0; e < E; ++e) out[c + e] = sg[i][e], out[H + c + e] = sb[i][e];
        }
    }
}

template <class T, int E, bool CK>
__global__ void __launch_bounds__(kNormThreads)
norm_bwd_block_kernel(const T *__restrict__ gy, int64_t ldg, NormSource src, const float2 *__restrict__ stats,
                      NormParam par, T *__restrict__ gx, int64_t ldgx, float *__restrict__ partials, int64_t n, int H)
{
    extern __shared__ float sums[];  // [2, H]: a column belongs to one thread
    __shared__ float red[kNormWarps];
    const float invH = 1.0f / (float)H;
    for (int c = threadIdx.x * E; c < H; c += kNormThreads * E) {
#pragma unroll
        for (int e = 0; e < E; ++e) sums[c + e] = sums[H + c + e] = 0.f;
    }
    for (int64_t r = blockIdx.x; r < n; r += gridDim.x) {
        const float2 st = __ldg(stats + r);
        const NormAffine f = norm_affine<CK>(src, r, st);
        float s1 = 0.f, s2 = 0.f, a[E], v[E], g[E];
        for (int c = threadIdx.x * E; c < H; c += kNormThreads * E) {
            load_row<T, E>(gy + r * ldg + c, a);
            load_source<T, E, CK>(src, r, c, v);
            load_param<T, E>(par.gamma, par.f32, c, 1.f, g);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float xh = norm_hat<CK>(v[e], f);
                sums[c + e] += a[e] * xh;
                sums[H + c + e] += a[e];
                s1 += a[e] * g[e];
                s2 += a[e] * g[e] * xh;
            }
        }
        const float m1 = block_sum(s1, red) * invH, m2 = block_sum(s2, red) * invH;
        for (int c = threadIdx.x * E; c < H; c += kNormThreads * E) {
            load_row<T, E>(gy + r * ldg + c, a);
            load_source<T, E, CK>(src, r, c, v);
            load_param<T, E>(par.gamma, par.f32, c, 1.f, g);
#pragma unroll
            for (int e = 0; e < E; ++e) a[e] = st.y * (a[e] * g[e] - m1 - norm_hat<CK>(v[e], f) * m2);
            store_row<T, E>(gx + r * ldgx + c, a);
        }
    }
    for (int c = threadIdx.x * E; c < H; c += kNormThreads * E) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            partials[(size_t)blockIdx.x * 2 * H + c + e] = sums[c + e];
            partials[(size_t)blockIdx.x * 2 * H + H + c + e] = sums[H + c + e];
        }
    }
}

// out[k] = sum over the blocks of partials[blocks, 2 H], in a fixed order: 32 columns a block, the partial rows dealt
// over its 32 warps, whose sums are added in turn
__global__ void __launch_bounds__(1024)
norm_reduce_kernel(const float *__restrict__ partials, int blocks, int H, void *__restrict__ g_gamma,
                   void *__restrict__ g_beta, int dtype)
{
    __shared__ float t[32][33];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int k = blockIdx.x * 32 + lane;
    float acc = 0.f;
    if (k < 2 * H) {
        for (int b = w; b < blocks; b += 32) acc += partials[(size_t)b * 2 * H + k];
    }
    t[w][lane] = acc;
    __syncthreads();
    if (w != 0 || k >= 2 * H) return;
    for (int i = 1; i < 32; ++i) acc += t[i][lane];
    void *out = k < H ? g_gamma : g_beta;
    const int c = k < H ? k : k - H;
    if (dtype == SGNN_F32) static_cast<float *>(out)[c] = acc;
    else if (dtype == SGNN_BF16) static_cast<__nv_bfloat16 *>(out)[c] = __float2bfloat16_rn(acc);
    else static_cast<__half *>(out)[c] = __float2half_rn(acc);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
struct NormCall {
    int dtype;
    const void *x;  // forward input, or the backward's source where there are no codes
    int64_t ldx;
    NormParam par;
    float eps;
    void *y;
    int64_t ldy;
    float2 *stats;
    uint8_t *codes;
    int64_t ldc;
    float2 *params;
    const void *gy;
    int64_t ldg;
    void *gx;
    int64_t ldgx;
    float *partials;
    int64_t n;
    int H;
    cudaStream_t stream;
};

static int norm_blocks_cap() { return sm_count() * 8; }

// Blocks of a call: enough for every warp (or block) to have a row, at most what is resident at once.
template <class K>
static int norm_grid(K kernel, int64_t n, int rows_per_block, size_t smem, size_t smem_cap, ResidentCache &cache, int *grid)
{
    int g = 0;
    int rc = resident_blocks(kernel, kNormThreads, smem, smem_cap, cache, &g);
    if (rc) return rc;
    if (g > norm_blocks_cap()) g = norm_blocks_cap();
    const int64_t need = ceil_div(n, rows_per_block);
    *grid = (int)(g < need ? g : need);
    return SGNN_OK;
}

template <class T, int E, int NV, bool CK, int LANES>
static int norm_fwd_launch(const NormCall &c)
{
    static ResidentCache cache;
    int grid = 0;
    if constexpr (NV > 0) {
        int rc = norm_grid(norm_fwd_warp_kernel<T, E, NV, CK, LANES>, c.n, kNormThreads / LANES, 0, 0, cache, &grid);
        if (rc) return rc;
        norm_fwd_warp_kernel<T, E, NV, CK, LANES><<<grid, kNormThreads, 0, c.stream>>>(
            static_cast<const T *>(c.x), c.ldx, c.par, c.eps, static_cast<T *>(c.y), c.ldy, c.stats, c.codes, c.ldc,
            c.params, c.n, c.H);
    } else {
        int rc = norm_grid(norm_fwd_block_kernel<T, E, CK>, c.n, 1, 0, 0, cache, &grid);
        if (rc) return rc;
        norm_fwd_block_kernel<T, E, CK><<<grid, kNormThreads, 0, c.stream>>>(
            static_cast<const T *>(c.x), c.ldx, c.par, c.eps, static_cast<T *>(c.y), c.ldy, c.stats, c.codes, c.ldc,
            c.params, c.n, c.H);
    }
    SGNN_LAUNCH_OK("layer norm forward");
    return SGNN_OK;
}

template <class T, int E, int NV, bool CK, int LANES>
static int norm_bwd_launch(const NormCall &c, int *blocks)
{
    static ResidentCache cache;
    const NormSource src{c.x, c.ldx, c.codes, c.ldc, c.params};
    if constexpr (NV > 0) {
        // room for the widest row of this kernel, whatever the row: the answer about residency then stays the same
        constexpr size_t most = (size_t)kNormWarps * 2 * LANES * E * NV * sizeof(float);
        const size_t smem = (size_t)kNormWarps * 2 * c.H * sizeof(float);
        int rc = norm_grid(norm_bwd_warp_kernel<T, E, NV, CK, LANES>, c.n, kNormThreads / LANES, E * NV <= 8 ? most : smem, most, cache, blocks);
        if (rc) return rc;
        norm_bwd_warp_kernel<T, E, NV, CK, LANES><<<*blocks, kNormThreads, smem, c.stream>>>(
            static_cast<const T *>(c.gy), c.ldg, src, c.stats, c.par, static_cast<T *>(c.gx), c.ldgx, c.partials, c.n,
            c.H);
    } else if constexpr (NV < 0) {
        int rc = norm_grid(norm_bwd_wide_kernel<T, E, CK>, c.n, 1, 0, 0, cache, blocks);
        if (rc) return rc;
        norm_bwd_wide_kernel<T, E, CK><<<*blocks, kNormThreads, 0, c.stream>>>(
            static_cast<const T *>(c.gy), c.ldg, src, c.stats, c.par, static_cast<T *>(c.gx), c.ldgx, c.partials, c.n,
            c.H);
    } else {
        const size_t smem = (size_t)2 * c.H * sizeof(float);
        int rc = norm_grid(norm_bwd_block_kernel<T, E, CK>, c.n, 1, smem, 2 * kNormMaxWidth * sizeof(float), cache, blocks);
        if (rc) return rc;
        norm_bwd_block_kernel<T, E, CK><<<*blocks, kNormThreads, smem, c.stream>>>(
            static_cast<const T *>(c.gy), c.ldg, src, c.stats, c.par, static_cast<T *>(c.gx), c.ldgx, c.partials, c.n,
            c.H);
    }
    SGNN_LAUNCH_OK("layer norm backward");
    return SGNN_OK;
}

// Staged rows: packed operands on 16-byte boundaries, rows of a whole warp's length (narrower ones share a warp: 600000 x 99 fp32
// 399 us staged, 263 so; 300000 x 201 239 us staged, 260 not); where narrow accesses were the alternative.
// The ring has as many buffers as leave room for two blocks an SM, at least two, at most four.
static bool norm_can_stage(const NormCall &c, size_t bytes)
{
    const bool fwd = c.y != nullptr;
    const auto packed = [&](const void *p, int64_t ld) { return ld == c.H && aligned16(p); };
    return c.n >= kNormWarps && c.H <= (fwd ? kStagedForward : bytes == 4 ? kNormSplit : 1024) && c.H > 128 && packed(c.x, c.ldx) &&
           (fwd ? packed(c.y, c.ldy) : packed(c.gy, c.ldg) && packed(c.gx, c.ldgx));
}
struct NormStage {
    size_t stride, second, smem;
    int depth;
};
static NormStage norm_stage(const NormCall &c, size_t bytes, int operands, int vectors)
{
    NormStage g{};
    const size_t one = ((size_t)kNormWarps * c.H * bytes + 127) / 128 * 128;
    const size_t head = ((size_t)vectors * c.H * sizeof(float) + 127) / 128 * 128;
    g.second = operands == 2 ? one : 0;
    g.stride = one * operands;
    g.depth = (int)((110 * 1024 - head) / g.stride);
    g.depth = g.depth < 2 ? 2 : g.depth > kStagedMax ? kStagedMax : g.depth;
    size_t ring = g.stride * g.depth;
    const size_t sums = 2 * (size_t)c.H * sizeof(float);
    if (ring < sums) ring = sums;
    g.smem = head + ring;
    return g;
}

template <class T, int E, int NV>
static int norm_fwd_staged(const NormCall &c)
{
    static ResidentCache cache;
    const NormStage g = norm_stage(c, sizeof(T), 1, 2);
    int grid = 0;
    int rc = norm_grid(norm_fwd_staged_kernel<T, E, NV>, c.n, kNormWarps, g.smem, kStagedCap, cache, &grid);
    if (rc) return rc;
    norm_fwd_staged_kernel<T, E, NV><<<grid, kNormThreads, g.smem, c.stream>>>(static_cast<const T *>(c.x), c.par, c.eps,
                                                                             static_cast<T *>(c.y), c.stats, c.n, c.H, g.stride, g.depth);
    SGNN_LAUNCH_OK("layer norm forward");
    return SGNN_OK;
}
template <class T, int E, int NV>
static int norm_bwd_staged(const NormCall &c, int *blocks)
{
    static ResidentCache cache;
    const NormStage g = norm_stage(c, sizeof(T), 2, 1);
    int rc = norm_grid(norm_bwd_staged_kernel<T, E, NV>, c.n, kNormWarps, g.smem, kStagedCap, cache, blocks);
    if (rc) return rc;
    norm_bwd_staged_kernel<T, E, NV><<<*blocks, kNormThreads, g.smem, c.stream>>>(
        static_cast<const T *>(c.gy), static_cast<const T *>(c.x), c.stats, c.par, static_cast<T *>(c.gx), c.partials, c.n, c.H, g.stride,
        g.second, g.depth);
    SGNN_LAUNCH_OK("layer norm backward");
    return SGNN_OK;
}
// 8, 12, 20 or 32 elements a lane, two at a time where 16-bit rows of even length allow it
#define SGNN_NORM_STAGED(FWD, T, fn, ...)                                                                                    \
    do {                                                                                                                \
        if constexpr (sizeof(T) == 2) {                                                                                 \
            if (c.H % 2 == 0) {                                                                                         \
                if (c.H <= 256) return fn<T, 2, 4>(c, ##__VA_ARGS__);                                                   \
                if (c.H <= 384) return fn<T, 2, 6>(c, ##__VA_ARGS__);                                                   \
                if (c.H <= 640) return fn<T, 2, 10>(c, ##__VA_ARGS__);                                                  \
                if (c.H <= 1024) return fn<T, 2, 16>(c, ##__VA_ARGS__);                                                 \
                return fn<T, 2, FWD ? 32 : 16>(c, ##__VA_ARGS__);                                                       \
            }                                                                                                           \
        }                                                                                                               \
        if (c.H <= 256) return fn<T, 1, 8>(c, ##__VA_ARGS__);                                                           \
        if (c.H <= 384) return fn<T, 1, 12>(c, ##__VA_ARGS__);                                                          \
        if (c.H <= 640) return fn<T, 1, 20>(c, ##__VA_ARGS__);                                                          \
        if (c.H <= 1024) return fn<T, 1, 32>(c, ##__VA_ARGS__);                                                         \
        return fn<T, 1, FWD ? 64 : 32>(c, ##__VA_ARGS__);                                                               \
    } while (0)

// fn<T, E, NV, CK, LANES>(c, ...) with the lanes of a row and the accesses a lane needs for it (NV = 0: the block kernel, -1:
// the backward's for rows up to kNormWide)
#define SGNN_NORM_NV(FWD, T, E, fn, ...)                                                                                     \
    do {                                                                                                                \
        const int lanes = row_lanes(c.H), need = (int)ceil_div(c.H, 32 * E);                                            \
        if (lanes == 4) return fn<T, E, 8 / E, CK, 4>(__VA_ARGS__);                                                     \
        if (lanes == 8) return fn<T, E, 8 / E, CK, 8>(__VA_ARGS__);                                                     \
        if (lanes == 16) return fn<T, E, 8 / E, CK, 16>(__VA_ARGS__);                                                   \
        if (need <= 8 / E) return fn<T, E, 8 / E, CK, 32>(__VA_ARGS__);                                                 \
        if constexpr (E >= 4) {                                                                                         \
            if (need <= 16 / E) return fn<T, E, 16 / E, CK, 32>(__VA_ARGS__);                                           \
        }                                                                                                               \
        if (!FWD && c.H > (CK && E != 4 ? 512 : kNormSplit) && c.H <= kNormWide) return fn<T, E, FWD ? 0 : -1, CK, 32>(__VA_ARGS__); \
        if constexpr (FWD || !CK || E != 8) {                                                                           \
            if (need <= 32 / E) return fn<T, E, 32 / E, CK, 32>(__VA_ARGS__);                                           \
        }                                                                                                               \
        if (FWD && E >= 4 && need <= 64 / E) return fn<T, E, FWD && E >= 4 ? 64 / E : 0, CK, 32>(__VA_ARGS__);          \
        return fn<T, E, 0, CK, 32>(__VA_ARGS__);                                                                        \
    } while (0)

template <bool CK>
static int norm_fwd_dispatch(const NormCall &c)
{
    const size_t b = elem_bytes(c.dtype);
    const int wide = (int)(16 / b);
    const size_t pb = c.par.f32 ? 4 : b;
    const RowOperand ops[] = {{c.x, c.ldx, b}, {c.y, c.ldy, b}, {c.par.gamma, 0, pb}, {c.par.beta, 0, pb},
                              {CK ? c.codes : nullptr, c.ldc, 1}};
    const int e = row_step(c.H, wide, ops);
    if (!CK && e != wide && norm_can_stage(c, b)) {
        if (c.dtype == SGNN_F32) SGNN_NORM_STAGED(true, float, norm_fwd_staged);
        if (c.dtype == SGNN_BF16) SGNN_NORM_STAGED(true, __nv_bfloat16, norm_fwd_staged);
        SGNN_NORM_STAGED(true, __half, norm_fwd_staged);
    }
    if (c.dtype == SGNN_F32) {
        if (e == 4) SGNN_NORM_NV(true, float, 4, norm_fwd_launch, c);
        if (e == 2) SGNN_NORM_NV(true, float, 2, norm_fwd_launch, c);
        SGNN_NORM_NV(true, float, 1, norm_fwd_launch, c);
    }
    if (c.dtype == SGNN_BF16) {
        if (e == 8) SGNN_NORM_NV(true, __nv_bfloat16, 8, norm_fwd_launch, c);
        if (e == 2) SGNN_NORM_NV(true, __nv_bfloat16, 2, norm_fwd_launch, c);
        SGNN_NORM_NV(true, __nv_bfloat16, 1, norm_fwd_launch, c);
    }
    if (e == 8) SGNN_NORM_NV(true, __half, 8, norm_fwd_launch, c);
    if (e == 2) SGNN_NORM_NV(true, __half, 2, norm_fwd_launch, c);
    SGNN_NORM_NV(true, __half, 1, norm_fwd_launch, c);
}

template <bool CK>
static int norm_bwd_dispatch(const NormCall &c, int *blocks)
{
    const size_t b = elem_bytes(c.dtype);
    const int wide = (int)(16 / b);
    const RowOperand ops[] = {{c.gy, c.ldg, b}, {c.gx, c.ldgx, b}, {c.par.gamma, 0, c.par.f32 ? 4 : b},
                              {CK ? nullptr : c.x, c.ldx, b}, {CK ? c.codes : nullptr, c.ldc, 1}};
    const int e = row_step(c.H, wide, ops);
    // Rows on boundaries that a lane cannot hold in eight elements are staged too: their column sums stay in registers
    // (600000 x 512 bf16: 464 us against 1254, 300000 x 512 fp32: 298 against 392), but for 32 fp32 elements a lane (150000 x 1024:
    // 607 us against 449).
    if (!CK && norm_can_stage(c, b) && (e != wide || (c.H > 256 && (b == 2 || c.H <= 640)))) {
        if (c.dtype == SGNN_F32) SGNN_NORM_STAGED(false, float, norm_bwd_staged, blocks);
        if (c.dtype == SGNN_BF16) SGNN_NORM_STAGED(false, __nv_bfloat16, norm_bwd_staged, blocks);
        SGNN_NORM_STAGED(false, __half, norm_bwd_staged, blocks);
    }
    if (c.dtype == SGNN_F32) {
        if (e == 4) SGNN_NORM_NV(false, float, 4, norm_bwd_launch, c, blocks);
        if (e == 2) SGNN_NORM_NV(false, float, 2, norm_bwd_launch, c, blocks);
        SGNN_NORM_NV(false, float, 1, norm_bwd_launch, c, blocks);
    }
    if (c.dtype == SGNN_BF16) {
        if (e == 8) SGNN_NORM_NV(false, __nv_bfloat16, 8, norm_bwd_launch, c, blocks);
        if (e == 2) SGNN_NORM_NV(false, __nv_bfloat16, 2, norm_bwd_launch, c, blocks);
        SGNN_NORM_NV(false, __nv_bfloat16, 1, norm_bwd_launch, c, blocks);
    }
    if (e == 8) SGNN_NORM_NV(false, __half, 8, norm_bwd_launch, c, blocks);
    if (e == 2) SGNN_NORM_NV(false, __half, 2, norm_bwd_launch, c, blocks);
    SGNN_NORM_NV(false, __half, 1, norm_bwd_launch, c, blocks);
}
#undef SGNN_NORM_NV
#undef SGNN_NORM_STAGED

static int norm_check(const char *who, int dtype, int param_dtype, int64_t n, int64_t H)
{
    SGNN_REQUIRE(elem_known(dtype) && elem_known(param_dtype), SGNN_ERR_INVALID_ARGUMENT, "%s: unknown element type", who);
    SGNN_REQUIRE(param_dtype == dtype || param_dtype == SGNN_F32, SGNN_ERR_INVALID_ARGUMENT,
                 "%s: gamma and beta must be fp32 or of the activation type", who);
    SGNN_REQUIRE(n >= 0 && H > 0, SGNN_ERR_INVALID_ARGUMENT, "%s: bad size", who);
    SGNN_REQUIRE(H <= kNormMaxWidth, SGNN_ERR_UNSUPPORTED, "%s: rows of at most %d elements (got %lld)", who,
                 kNormMaxWidth, (long long)H);
    SGNN_REQUIRE(n <= (1LL << 40), SGNN_ERR_TOO_LARGE, "%s: too many rows", who);
    return SGNN_OK;
}

static bool aligned_to(const void *p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

}  // namespace sgnn

using namespace sgnn;

extern "C" SGNN_API int sgnn_layer_norm_forward(int dtype, const void *d_x, int64_t ldx, int param_dtype,
                                                const void *d_gamma, const void *d_beta, float eps, void *d_y,
                                                int64_t ldy, float *d_stats, uint8_t *d_codes, int64_t ldc,
                                                float *d_params, int64_t n, int64_t H, void *stream)
{
    const char *who = "layer_norm_forward";
    int rc = norm_check(who, dtype, param_dtype, n, H);
    if (rc) return rc;
    SGNN_REQUIRE(eps >= 0.f, SGNN_ERR_INVALID_ARGUMENT, "%s: eps must not be negative", who);
    if (n == 0) return SGNN_OK;
    SGNN_REQUIRE(d_x && d_y && d_stats, SGNN_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
    SGNN_REQUIRE((d_codes == nullptr) == (d_params == nullptr), SGNN_ERR_INVALID_ARGUMENT,
                 "%s: codes and params belong together", who);
    SGNN_REQUIRE((n == 1 || (ldx >= H && ldy >= H)) && (d_codes == nullptr || n == 1 || ldc >= H), SGNN_ERR_INVALID_ARGUMENT,
                 "%s: leading dimension shorter than a row", who);
    const size_t b = elem_bytes(dtype), pb = elem_bytes(param_dtype);
    SGNN_REQUIRE(aligned_to(d_x, b) && aligned_to(d_y, b) && aligned_to(d_gamma, pb) && aligned_to(d_beta, pb) &&
                     aligned_to(d_stats, 8) && aligned_to(d_params, 8),
                 SGNN_ERR_INVALID_ARGUMENT, "%s: pointers must be aligned to their element (stats, params: 8 bytes)", who);
    NormCall c{};
    c.dtype = dtype, c.x = d_x, c.ldx = ldx, c.par = NormParam{d_gamma, d_beta, param_dtype == SGNN_F32}, c.eps = eps;
    c.y = d_y, c.ldy = ldy, c.stats = reinterpret_cast<float2 *>(d_stats), c.codes = d_codes, c.ldc = ldc;
    c.params = reinterpret_cast<float2 *>(d_params), c.n = n, c.H = (int)H, c.stream = (cudaStream_t)stream;
    return d_codes ? norm_fwd_dispatch<true>(c) : norm_fwd_dispatch<false>(c);
}

extern "C" SGNN_API int sgnn_layer_norm_blocks(void) { return norm_blocks_cap(); }

extern "C" SGNN_API int sgnn_layer_norm_backward(int dtype, const void *d_gy, int64_t ldg, const void *d_x, int64_t ldx,
                                                 const uint8_t *d_codes, int64_t ldc, const float *d_params,
                                                 const float *d_stats, int param_dtype, const void *d_gamma,
                                                 void *d_gx, int64_t ldgx, void *d_g_gamma, void *d_g_beta,
                                                 float *d_partials, int64_t n, int64_t H, void *stream)
{
    const char *who = "layer_norm_backward";
    int rc = norm_check(who, dtype, param_dtype, n, H);
    if (rc) return rc;
    SGNN_REQUIRE(d_g_gamma && d_g_beta, SGNN_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
    const size_t b = elem_bytes(dtype), pb = elem_bytes(param_dtype);
    cudaStream_t s = (cudaStream_t)stream;
    if (n == 0) {
        SGNN_CUDA_OK(cudaMemsetAsync(d_g_gamma, 0, (size_t)H * pb, s));
        SGNN_CUDA_OK(cudaMemsetAsync(d_g_beta, 0, (size_t)H * pb, s));
        return SGNN_OK;
    }
    SGNN_REQUIRE(d_gy && d_gx && d_stats && d_partials, SGNN_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
    SGNN_REQUIRE((d_codes == nullptr) == (d_params == nullptr) && (d_codes == nullptr) != (d_x == nullptr),
                 SGNN_ERR_INVALID_ARGUMENT, "%s: exactly one of x and (codes, params) must be given", who);
    SGNN_REQUIRE(n == 1 || (ldg >= H && ldgx >= H && (d_x == nullptr || ldx >= H) && (d_codes == nullptr || ldc >= H)),
                 SGNN_ERR_INVALID_ARGUMENT, "%s: leading dimension shorter than a row", who);
    SGNN_REQUIRE(aligned_to(d_gy, b) && aligned_to(d_x, b) && aligned_to(d_gx, b) && aligned_to(d_gamma, pb) &&
                     aligned_to(d_g_gamma, pb) && aligned_to(d_g_beta, pb) && aligned_to(d_stats, 8) &&
                     aligned_to(d_params, 8) && aligned_to(d_partials, 4),
                 SGNN_ERR_INVALID_ARGUMENT, "%s: pointers must be aligned to their element (stats, params: 8 bytes)", who);
    NormCall c{};
    c.dtype = dtype, c.gy = d_gy, c.ldg = ldg, c.x = d_x, c.ldx = ldx;
    c.codes = const_cast<uint8_t *>(d_codes), c.ldc = ldc;
    c.params = reinterpret_cast<float2 *>(const_cast<float *>(d_params));
    c.stats = reinterpret_cast<float2 *>(const_cast<float *>(d_stats));
    c.par = NormParam{d_gamma, nullptr, param_dtype == SGNN_F32}, c.gx = d_gx, c.ldgx = ldgx, c.partials = d_partials;
    c.n = n, c.H = (int)H, c.stream = s;
    int blocks = 0;
    rc = d_codes ? norm_bwd_dispatch<true>(c, &blocks) : norm_bwd_dispatch<false>(c, &blocks);
    if (rc) return rc;
    norm_reduce_kernel<<<(int)ceil_div(2 * H, 32), 1024, 0, s>>>(d_partials, blocks, (int)H, d_g_gamma, d_g_beta,
                                                                 param_dtype);
    SGNN_LAUNCH_OK("layer norm column sums");
    return SGNN_OK;
}
