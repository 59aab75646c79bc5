// Activation checkpoints in 8 bits (sm_100a): what a layer keeps of its input for the backward pass, one byte an
// element and two fp32 numbers a row in place of four bytes an element.
//
//     zp = min of the row, sc = (max - min) / 255, code = rne((x - zp) / sc);  restored value = zp + sc code
//
// The quantiser is the boundary exchange's (8 bits, min-max a row), for rows of any width, strided, in fp32, bf16 or
// fp16.  See row_io.cuh for rows without a range and for NaN and infinities.  Both kernels are bound by memory: the row
// is read once (rows of up to 2048 elements, 1024 where they allow no accesses of 16 bytes, stay in a warp's registers, several narrow
// ones at a time; longer ones are read a second time from L1 / L2 by the block that owns them).
#include "row_io.cuh"

namespace sgnn {

constexpr int kCkptThreads = 256;
constexpr int kCkptWarps = kCkptThreads / 32;

template <class T, int E, int NV, int LANES>
__global__ void __launch_bounds__(kCkptThreads)
checkpoint_pack_warp_kernel(const T *__restrict__ x, int64_t ldx, uint8_t *__restrict__ codes, int64_t ldc,
                            float2 *__restrict__ params, int64_t n, int F)
{
    constexpr int kRows = 32 / LANES;  // of a warp at a time
    const int lane = threadIdx.x % LANES, sub = (threadIdx.x & 31) / LANES;
    const int64_t step = (int64_t)gridDim.x * kCkptWarps * kRows;
    for (int64_t r0 = ((int64_t)blockIdx.x * kCkptWarps + (threadIdx.x >> 5)) * kRows; r0 < n; r0 += step) {
        const int64_t r = r0 + sub;
        const int width = r < n ? F : 0;
        float v[NV][E];
        float mn = INFINITY, mx = -INFINITY, poison = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (lane + LANES * i) * E;
            if (c < width) load_row<T, E>(x + r * ldx + c, v[i]);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if ((lane + LANES * i) * E < width) {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    mn = fminf(mn, v[i][e]), mx = fmaxf(mx, v[i][e]), poison = __fmaf_rn(v[i][e], 0.f, poison);
            }
        }
        const RowQ q = row_quantiser(row_min<LANES>(mn), row_max<LANES>(mx), row_sum<LANES>(poison));
        if (lane == 0 && r < n) params[r] = make_float2(q.mn, q.sc);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (lane + LANES * i) * E;
            if (c < width) store_codes<E>(codes + r * ldc + c, v[i], q);
        }
    }
}

template <class T, int E>
__global__ void __launch_bounds__(kCkptThreads)
checkpoint_pack_block_kernel(const T *__restrict__ x, int64_t ldx, uint8_t *__restrict__ codes, int64_t ldc,
                             float2 *__restrict__ params, int64_t n, int F)
{
    __shared__ float red[3][kCkptWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int64_t r = blockIdx.x; r < n; r += gridDim.x) {
        const T *xr = x + r * ldx;
        float mn = INFINITY, mx = -INFINITY, poison = 0.f, v[E];
        for (int c = threadIdx.x * E; c < F; c += kCkptThreads * E) {
            load_row<T, E>(xr + c, v);
#pragma unroll
            for (int e = 0; e < E; ++e) mn = fminf(mn, v[e]), mx = fmaxf(mx, v[e]), poison = __fmaf_rn(v[e], 0.f, poison);
        }
        mn = redux_min(mn), mx = redux_max(mx), poison = all_sum(poison);
        __syncthreads();  // the sums of the row before are read
        if (lane == 0) red[0][warp] = mn, red[1][warp] = mx, red[2][warp] = poison;
        __syncthreads();
        mn = INFINITY, mx = -INFINITY, poison = 0.f;
#pragma unroll
        for (int w = 0; w < kCkptWarps; ++w) mn = fminf(mn, red[0][w]), mx = fmaxf(mx, red[1][w]), poison += red[2][w];
        const RowQ q = row_quantiser(mn, mx, poison);
        if (threadIdx.x == 0) params[r] = make_float2(q.mn, q.sc);
        for (int c = threadIdx.x * E; c < F; c += kCkptThreads * E) {
            load_row<T, E>(xr + c, v);
            store_codes<E>(codes + r * ldc + c, v, q);
        }
    }
}

template <class T, int E, int LANES>
__global__ void __launch_bounds__(kCkptThreads)
checkpoint_unpack_kernel(const uint8_t *__restrict__ codes, int64_t ldc, const float2 *__restrict__ params,
                         T *__restrict__ out, int64_t ldo, int64_t n, int F)
{
    constexpr int kRows = kCkptThreads / LANES;  // of a block at a time
    const int lane = threadIdx.x % LANES;
    const int64_t step = (int64_t)gridDim.x * kRows;
    for (int64_t r = (int64_t)blockIdx.x * kRows + threadIdx.x / LANES; r < n; r += step) {
        const float2 p = __ldg(params + r);
        for (int c = lane * E; c < F; c += LANES * E) {
            float v[E];
            load_codes<E>(codes + r * ldc + c, v);
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = __fmaf_rn(v[e], p.y, p.x);
            store_row<T, E>(out + r * ldo + c, v);
        }
    }
}

struct CkptCall {
    int dtype;
    void *x;  // read by pack, written by unpack
    int64_t ldx;
    uint8_t *codes;
    int64_t ldc;
    float2 *params;
    int64_t n;
    int F;
    cudaStream_t stream;
};

template <class K>
static int ckpt_grid(K kernel, int64_t n, int rows_per_block, ResidentCache &cache, int *grid)
{
    int g = 0;
    int rc = resident_blocks(kernel, kCkptThreads, 0, 0, cache, &g);
    const int64_t need = ceil_div(n, rows_per_block);
    *grid = (int)(g < need ? g : need);
    return rc;
}

template <class T, int E, int NV, int LANES>
static int pack_launch(const CkptCall &c)
{
    static ResidentCache cache;
    int grid = 0, rc;
    if constexpr (NV > 0) {
        if ((rc = ckpt_grid(checkpoint_pack_warp_kernel<T, E, NV, LANES>, c.n, kCkptThreads / LANES, cache, &grid))) return rc;
        checkpoint_pack_warp_kernel<T, E, NV, LANES><<<grid, kCkptThreads, 0, c.stream>>>(static_cast<const T *>(c.x), c.ldx,
                                                                                   c.codes, c.ldc, c.params, c.n, c.F);
    } else {
        if ((rc = ckpt_grid(checkpoint_pack_block_kernel<T, E>, c.n, 1, cache, &grid))) return rc;
        checkpoint_pack_block_kernel<T, E><<<grid, kCkptThreads, 0, c.stream>>>(static_cast<const T *>(c.x), c.ldx,
                                                                                c.codes, c.ldc, c.params, c.n, c.F);
    }
    SGNN_LAUNCH_OK("checkpoint_pack_rows");
    return SGNN_OK;
}

template <class T, int E>
static int pack_width(const CkptCall &c)
{
    const int lanes = row_lanes(c.F), need = (int)ceil_div(c.F, 32 * E);
    if (lanes == 4) return pack_launch<T, E, 8 / E, 4>(c);
    if (lanes == 8) return pack_launch<T, E, 8 / E, 8>(c);
    if (lanes == 16) return pack_launch<T, E, 8 / E, 16>(c);
    if (need <= 8 / E) return pack_launch<T, E, 8 / E, 32>(c);
    if constexpr (E >= 4) {
        if (need <= 16 / E) return pack_launch<T, E, 16 / E, 32>(c);
    }
    if (need <= 32 / E) return pack_launch<T, E, 32 / E, 32>(c);
    if constexpr (E >= 4) {
        if (need <= 64 / E) return pack_launch<T, E, 64 / E, 32>(c);
    }
    return pack_launch<T, E, 0, 32>(c);
}

template <class T, int E, int LANES>
static int unpack_launch(const CkptCall &c)
{
    static ResidentCache cache;
    int grid = 0;
    int rc = ckpt_grid(checkpoint_unpack_kernel<T, E, LANES>, c.n, kCkptThreads / LANES, cache, &grid);
    if (rc) return rc;
    checkpoint_unpack_kernel<T, E, LANES><<<grid, kCkptThreads, 0, c.stream>>>(c.codes, c.ldc, c.params, static_cast<T *>(c.x),
                                                                        c.ldx, c.n, c.F);
    SGNN_LAUNCH_OK("checkpoint_unpack_rows");
    return SGNN_OK;
}

template <class T, int E>
static int unpack_width(const CkptCall &c)
{
    const int lanes = row_lanes(c.F);
    if (lanes == 4) return unpack_launch<T, E, 4>(c);
    if (lanes == 8) return unpack_launch<T, E, 8>(c);
    if (lanes == 16) return unpack_launch<T, E, 16>(c);
    return unpack_launch<T, E, 32>(c);
}

template <class T, bool PACK>
static int ckpt_step(const CkptCall &c)
{
    constexpr int W = 16 / sizeof(T);
    const RowOperand ops[] = {{c.x, c.ldx, sizeof(T)}, {c.codes, c.ldc, 1}};
    const int e = row_step(c.F, W, ops);
    if constexpr (PACK) {
        if (e == W) return pack_width<T, W>(c);
        if (e == 2) return pack_width<T, 2>(c);
        return pack_width<T, 1>(c);
    } else {
        if (e == W) return unpack_width<T, W>(c);
        if (e == 2) return unpack_width<T, 2>(c);
        return unpack_width<T, 1>(c);
    }
}

template <bool PACK>
static int ckpt_run(const char *who, int dtype, const void *x, int64_t ldx, const uint8_t *codes, int64_t ldc,
                    const float *params, int64_t n, int64_t F, void *stream)
{
    SGNN_REQUIRE(elem_known(dtype), SGNN_ERR_INVALID_ARGUMENT, "%s: unknown element type", who);
    SGNN_REQUIRE(n >= 0 && F > 0, SGNN_ERR_INVALID_ARGUMENT, "%s: bad size", who);
    SGNN_REQUIRE(n <= (1LL << 40) && F < (1LL << 30), SGNN_ERR_TOO_LARGE, "%s: too large", who);
    if (n == 0) return SGNN_OK;
    SGNN_REQUIRE(x && codes && params, SGNN_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
    SGNN_REQUIRE(n == 1 || (ldx >= F && ldc >= F), SGNN_ERR_INVALID_ARGUMENT, "%s: leading dimension shorter than a row", who);
    SGNN_REQUIRE(reinterpret_cast<uintptr_t>(x) % elem_bytes(dtype) == 0 && reinterpret_cast<uintptr_t>(params) % 8 == 0,
                 SGNN_ERR_INVALID_ARGUMENT, "%s: pointers must be aligned to their element (params: 8 bytes)", who);
    const CkptCall c{dtype, const_cast<void *>(x), ldx, const_cast<uint8_t *>(codes), ldc,
                     reinterpret_cast<float2 *>(const_cast<float *>(params)), n, (int)F, (cudaStream_t)stream};
    if (dtype == SGNN_F32) return ckpt_step<float, PACK>(c);
    if (dtype == SGNN_BF16) return ckpt_step<__nv_bfloat16, PACK>(c);
    return ckpt_step<__half, PACK>(c);
}

}  // namespace sgnn

using namespace sgnn;

extern "C" SGNN_API int sgnn_checkpoint_pack_rows(int dtype, const void *d_x, int64_t ldx, uint8_t *d_codes, int64_t ldc,
                                                  float *d_params, int64_t n, int64_t F, void *stream)
{
    return ckpt_run<true>("checkpoint_pack_rows", dtype, d_x, ldx, d_codes, ldc, d_params, n, F, stream);
}

extern "C" SGNN_API int sgnn_checkpoint_unpack_rows(const uint8_t *d_codes, int64_t ldc, const float *d_params, int dtype,
                                                    void *d_out, int64_t ldo, int64_t n, int64_t F, void *stream)
{
    return ckpt_run<false>("checkpoint_unpack_rows", dtype, d_out, ldo, d_codes, ldc, d_params, n, F, stream);
}
