// Weight gradient of a linear map whose input was kept as 8-bit codes (sm_100a):
//
//     gW[m, k] = sum_r g[r, m] (zp_r + sc_r code[r, k])  (+ beta gW[m, k])
//
// The rows are split over the blocks; the partial products are added in a fixed order.
#include "row_io.cuh"
#include "tile_product.cuh"

namespace sgnn {

template <class T>
struct GradOperand {  // A(m, r) = g[r, m]
    const T *g;
    int64_t ldg;
    int M;
    __device__ float operator()(int64_t m, int64_t r) const { return m < M ? to_f32<T>(g[r * ldg + m]) : 0.f; }
};

struct CodeOperand {  // B(k, r) = zp_r + sc_r code[r, k]
    const uint8_t *codes;
    int64_t ldc;
    const float2 *params;
    int F;
    __device__ float operator()(int64_t k, int64_t r) const
    {
        return k < F ? __fmaf_rn((float)codes[r * ldc + k], params[r].y, params[r].x) : 0.f;
    }
};

struct PartialStore {
    float *out;
    int M, F;
    __device__ void operator()(int64_t m, int64_t n, const float (&acc)[4][4], int split) const
    {
        for (int i = 0; i < 4; ++i)
            for (int j = 0; j < 4; ++j)
                if (m + i < M && n + j < F) out[((int64_t)split * M + m + i) * F + n + j] = acc[i][j];
    }
};

__global__ void weight_grad_join_kernel(const float *__restrict__ partials, int splits, int M, int F, float beta,
                                        float *__restrict__ out, int64_t ldo)
{
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (int64_t)M * F) return;
    float acc = 0.f;
    for (int s = 0; s < splits; ++s) acc += partials[(int64_t)s * M * F + i];
    float *o = out + (i / F) * ldo + i % F;
    *o = beta == 0.f ? acc : acc + beta * *o;
}

static int weight_grad_splits(int64_t n, int64_t M, int64_t F)
{
    const int64_t tiles = ceil_div(M, kTile) * ceil_div(F, kTile), most = ceil_div(n, 256);
    int64_t s = ceil_div(4 * sm_count(), tiles);
    s = s < most ? s : most;
    return (int)(s < 1 ? 1 : s);
}

template <class T>
static int weight_grad_run(const void *g, int64_t ldg, const uint8_t *codes, int64_t ldc, const float2 *params, int64_t n,
                           int M, int F, float beta, float *out, int64_t ldo, float *partials, cudaStream_t s)
{
    const int splits = weight_grad_splits(n, M, F);
    const dim3 grid((unsigned)ceil_div(F, kTile), (unsigned)ceil_div(M, kTile), (unsigned)splits);
    tile_product_kernel<<<grid, kTileThreads, 0, s>>>(GradOperand<T>{static_cast<const T *>(g), ldg, M},
                                                      CodeOperand{codes, ldc, params, F}, PartialStore{partials, M, F}, n,
                                                      ceil_div(n, splits));
    SGNN_LAUNCH_OK("checkpoint_weight_grad");
    weight_grad_join_kernel<<<(unsigned)ceil_div((int64_t)M * F, 256), 256, 0, s>>>(partials, splits, M, F, beta, out, ldo);
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
    *bytes = n == 0 ? 0 : (size_t)weight_grad_splits(n, M, F) * M * F * sizeof(float);
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
    SGNN_REQUIRE(d_out != nullptr && ldo >= F, SGNN_ERR_INVALID_ARGUMENT, "%s: bad output", who);
    cudaStream_t s = (cudaStream_t)stream;
    if (n == 0) {
        weight_grad_join_kernel<<<(unsigned)ceil_div(M * F, 256), 256, 0, s>>>(nullptr, 0, (int)M, (int)F, beta, d_out, ldo);
        SGNN_LAUNCH_OK("checkpoint_weight_grad join");
        return SGNN_OK;
    }
    SGNN_REQUIRE(d_g && d_codes && d_params, SGNN_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
    SGNN_REQUIRE(n == 1 || (ldg >= M && ldc >= F), SGNN_ERR_INVALID_ARGUMENT, "%s: leading dimension shorter than a row", who);
    SGNN_REQUIRE(reinterpret_cast<uintptr_t>(d_g) % elem_bytes(dtype) == 0 && reinterpret_cast<uintptr_t>(d_params) % 8 == 0,
                 SGNN_ERR_INVALID_ARGUMENT, "%s: pointers must be aligned to their element (params: 8 bytes)", who);
    size_t need = 0;
    rc = sgnn_checkpoint_weight_grad_workspace_bytes(dtype, n, M, F, &need);
    if (rc) return rc;
    SGNN_REQUIRE(d_workspace != nullptr && workspace_bytes >= need, SGNN_ERR_WORKSPACE,
                 "%s: workspace of %zu bytes needed, %zu given", who, need, workspace_bytes);
    const float2 *params = reinterpret_cast<const float2 *>(d_params);
    float *partials = static_cast<float *>(d_workspace);
    if (dtype == SGNN_F32)
        return weight_grad_run<float>(d_g, ldg, d_codes, ldc, params, n, (int)M, (int)F, beta, d_out, ldo, partials, s);
    if (dtype == SGNN_BF16)
        return weight_grad_run<__nv_bfloat16>(d_g, ldg, d_codes, ldc, params, n, (int)M, (int)F, beta, d_out, ldo, partials, s);
    return weight_grad_run<__half>(d_g, ldg, d_codes, ldc, params, n, (int)M, (int)F, beta, d_out, ldo, partials, s);
}
