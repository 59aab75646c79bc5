// Negative log-likelihood of a linear classifier over many classes and its gradients (sm_100a), in pieces of the
// classes, so that the logits z = x W^T + b, [n, C], are never kept:
//
//     lse[r] = log sum_c exp z[r, c]        running maximum and sum over the pieces
//     loss   = inv_count sum_r (lse[r] - z[r, label])
//     G      = inv_count (exp(z - lse) - onehot)  piece by piece, from logits computed a second time
//     gx += G W_piece,  gw_piece = G^T x,  gb_piece = sum_r G
//
// The rows in the loss are listed first (in order); everything else works on the list, so that a row outside the mask
// costs nothing and whatever it holds is not read.
#include "row_io.cuh"
#include "tile_product.cuh"

namespace sgnn {

constexpr int kListRows = 2048;  // rows a block of the listing kernels looks at
constexpr int kListThreads = 256;

__device__ __forceinline__ bool in_loss(const int64_t *labels, const uint8_t *mask, int64_t r, int64_t n, int64_t C)
{
    if (r >= n || (mask != nullptr && mask[r] == 0)) return false;
    const int64_t l = labels[r];
    return l >= 0 && l < C;
}

__global__ void __launch_bounds__(kListThreads)
nll_count_kernel(const int64_t *__restrict__ labels, const uint8_t *__restrict__ mask, int64_t n, int64_t C, int *__restrict__ counts)
{
    int c = 0;
    for (int i = 0; i < kListRows / kListThreads; ++i)
        c += __syncthreads_count(in_loss(labels, mask, (int64_t)blockIdx.x * kListRows + i * kListThreads + threadIdx.x, n, C));
    if (threadIdx.x == 0) counts[blockIdx.x] = c;
}

// rows[0 .. m) = the rows in the loss, ascending; *total = m
__global__ void __launch_bounds__(kListThreads)
nll_list_kernel(const int64_t *__restrict__ labels, const uint8_t *__restrict__ mask, int64_t n, int64_t C,
                const int *__restrict__ counts, int *__restrict__ rows, int *__restrict__ total)
{
    __shared__ int part[kListThreads / 32], before[kListThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int s = 0;
    for (int b = threadIdx.x; b < blockIdx.x; b += kListThreads) s += counts[b];
    s = __reduce_add_sync(FULL, s);
    if (lane == 0) part[warp] = s;
    __syncthreads();
    int at = 0;
    for (int w = 0; w < kListThreads / 32; ++w) at += part[w];
    for (int i = 0; i < kListRows / kListThreads; ++i) {
        const int64_t r = (int64_t)blockIdx.x * kListRows + i * kListThreads + threadIdx.x;
        const bool on = in_loss(labels, mask, r, n, C);
        const unsigned vote = __ballot_sync(FULL, on);
        __syncthreads();
        if (lane == 0) before[warp] = __popc(vote);
        __syncthreads();
        int pos = at + __popc(vote & ((1u << lane) - 1u));
        for (int w = 0; w < kListThreads / 32; ++w) {
            if (w < warp) pos += before[w];
            at += before[w];
        }
        if (on) rows[pos] = (int)r;
    }
    if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) *total = at;
}

template <class T>
struct RowsOperand {  // A(i, k) = x[rows[i], k] of the listed rows
    const T *x;
    int64_t ldx;
    const int *rows, *total;
    int K;
    __device__ float operator()(int64_t i, int64_t k) const { return i < *total && k < K ? to_f32<T>(x[rows[i] * ldx + k]) : 0.f; }
};
template <class T>
struct RowsOperandT {  // B(k, i) = x[rows[i], k]
    RowsOperand<T> a;
    __device__ float operator()(int64_t k, int64_t i) const { return a(i, k); }
};
template <class T>
struct WeightOperand {  // B(c, k) = W[first + c, k]
    const T *w;
    int64_t ldw, first, C;
    int K;
    __device__ float operator()(int64_t c, int64_t k) const { return first + c < C && k < K ? to_f32<T>(w[(first + c) * ldw + k]) : 0.f; }
};
template <class T>
struct WeightOperandT {  // B(k, c) = W[first + c, k]
    WeightOperand<T> w;
    __device__ float operator()(int64_t k, int64_t c) const { return w(c, k); }
};
struct PieceOperand {  // A(i, c) = piece[i, c]
    const float *piece;
    int64_t width;
    const int *total;
    __device__ float operator()(int64_t i, int64_t c) const { return i < *total && c < width ? piece[i * width + c] : 0.f; }
};
struct PieceOperandT {  // A(c, i) = piece[i, c]
    PieceOperand p;
    __device__ float operator()(int64_t c, int64_t i) const { return p(i, c); }
};
struct PieceStore {
    float *piece;
    int64_t width;
    const int *total;
    __device__ void operator()(int64_t m, int64_t n, const float (&acc)[4][4], int) const
    {
        for (int i = 0; i < 4; ++i)
            for (int j = 0; j < 4; ++j)
                if (m + i < *total && n + j < width) piece[(m + i) * width + n + j] = acc[i][j];
    }
};
struct AddRows {  // gx accumulator of the listed rows
    float *out;
    int K;
    const int *total;
    __device__ void operator()(int64_t m, int64_t n, const float (&acc)[4][4], int) const
    {
        for (int i = 0; i < 4; ++i)
            for (int j = 0; j < 4; ++j)
                if (m + i < *total && n + j < K) out[(m + i) * K + n + j] += acc[i][j];
    }
};
template <class T>
struct WeightStore {
    T *out;
    int64_t ld, first, width;
    int K;
    float scale;
    __device__ void operator()(int64_t m, int64_t n, const float (&acc)[4][4], int) const
    {
        for (int i = 0; i < 4; ++i)
            for (int j = 0; j < 4; ++j)
                if (m + i < width && n + j < K) out[(first + m + i) * ld + n + j] = from_f32<T>(acc[i][j] * scale);
    }
};

struct NllBias {
    const void *b;
    bool f32;
};
template <class T>
__device__ __forceinline__ float bias_at(NllBias b, int64_t c)
{
    return b.b == nullptr ? 0.f : b.f32 ? static_cast<const float *>(b.b)[c] : to_f32<T>(static_cast<const T *>(b.b)[c]);
}

// running (maximum, sum of exp) of a row and its label's logit, one block a listed row
template <class T>
__global__ void __launch_bounds__(256)
nll_stats_kernel(const float *__restrict__ piece, int64_t first, int64_t width, NllBias bias, const int64_t *__restrict__ labels,
                 const int *__restrict__ rows, const int *__restrict__ total, float2 *__restrict__ run, float *__restrict__ picked)
{
    __shared__ float red[8];
    const int i = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (i >= *total) return;
    const int64_t label = labels[rows[i]] - first;
    float mx = -INFINITY;
    for (int64_t c = threadIdx.x; c < width; c += 256) mx = fmaxf(mx, piece[i * width + c] + bias_at<T>(bias, first + c));
    mx = warp_max(mx);
    if (lane == 0) red[warp] = mx;
    __syncthreads();
    float2 old = first == 0 ? make_float2(-INFINITY, 0.f) : run[i];
    for (int w = 0; w < 8; ++w) mx = fmaxf(mx, red[w]);
    mx = fmaxf(mx, old.x);
    const float ref = mx == -INFINITY ? 0.f : mx;  // a row of -inf so far
    __syncthreads();
    float s = 0.f;
    for (int64_t c = threadIdx.x; c < width; c += 256) {
        const float z = piece[i * width + c] + bias_at<T>(bias, first + c);
        s += expf(z - ref);
        if (c == label) picked[i] = z;
    }
    s = all_sum(s);
    if (lane == 0) red[warp] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = old.y * expf(old.x - ref);
        for (int w = 0; w < 8; ++w) s += red[w];
        run[i] = make_float2(mx, s);
    }
}

__global__ void nll_lse_kernel(const float2 *__restrict__ run, const int *__restrict__ rows, const int *__restrict__ total,
                               float *__restrict__ lse, float *__restrict__ lse_out)
{
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= *total) return;
    const float l = run[i].x + logf(run[i].y);
    lse[i] = l;
    if (lse_out) lse_out[rows[i]] = l;
}

__global__ void __launch_bounds__(1024)
nll_loss_kernel(const float *__restrict__ lse, const float *__restrict__ picked, const int *__restrict__ total, float inv_count,
                float *__restrict__ loss)
{
    __shared__ float red[32];
    float s = 0.f;
    for (int i = threadIdx.x; i < *total; i += 1024) s += lse[i] - picked[i];
    s = all_sum(s);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x < 32) {
        s = all_sum(red[threadIdx.x]);
        if (threadIdx.x == 0) *loss = s * inv_count;
    }
}

// piece of logits -> piece of exp(z - lse) - onehot
template <class T>
__global__ void __launch_bounds__(256)
nll_piece_grad_kernel(float *__restrict__ piece, int64_t first, int64_t width, NllBias bias, const int64_t *__restrict__ labels,
                      const int *__restrict__ rows, const int *__restrict__ total, const float *__restrict__ lse)
{
    const int i = blockIdx.x;
    if (i >= *total) return;
    const int64_t label = labels[rows[i]] - first;
    for (int64_t c = threadIdx.x; c < width; c += 256)
        piece[i * width + c] = expf(piece[i * width + c] + bias_at<T>(bias, first + c) - lse[i]) - (c == label ? 1.f : 0.f);
}

template <class T>
__global__ void nll_bias_grad_kernel(const float *__restrict__ piece, int64_t first, int64_t width, const int *__restrict__ total,
                                     float scale, bool f32, void *__restrict__ gb)
{
    const int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= width) return;
    float s = 0.f;
    for (int64_t i = 0; i < *total; ++i) s += piece[i * width + c];
    if (f32) static_cast<float *>(gb)[first + c] = s * scale;
    else static_cast<T *>(gb)[first + c] = from_f32<T>(s * scale);
}

template <class T>
__global__ void nll_rows_out_kernel(const float *__restrict__ acc, const int *__restrict__ rows, const int *__restrict__ total,
                                    float scale, T *__restrict__ gx, int64_t ldgx, int K)
{
    const int i = blockIdx.x;
    if (i >= *total) return;
    for (int k = threadIdx.x; k < K; k += blockDim.x) gx[rows[i] * ldgx + k] = from_f32<T>(acc[(int64_t)i * K + k] * scale);
}

struct NllSizes {
    int64_t blocks, width;  // listing blocks, classes of a piece
    size_t counts, rows, total, run, picked, lse, acc, piece, bytes;
};

static NllSizes nll_sizes(int64_t n, int64_t K, int64_t C, bool grad)
{
    NllSizes z{};
    z.blocks = ceil_div(n, kListRows);
    z.width = (64ll << 20) / (n * 4) / 64 * 64;
    if (z.width < 64) z.width = 64;
    if (z.width > C) z.width = C;
    size_t at = 0;
    const auto take = [&at](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    z.counts = take(z.blocks * 4), z.rows = take(n * 4), z.total = take(4), z.run = take(n * 8), z.picked = take(n * 4);
    z.lse = take(n * 4), z.acc = take(grad ? n * K * 4 : 0), z.piece = take(n * z.width * 4);
    z.bytes = at;
    return z;
}

static int nll_check(const char *who, int dtype, int64_t n, int64_t K, int64_t C)
{
    SGNN_REQUIRE(dtype == SGNN_F32 || dtype == SGNN_BF16, SGNN_ERR_INVALID_ARGUMENT, "%s: fp32 or bf16 only", who);
    SGNN_REQUIRE(n >= 0 && K > 0 && C > 0, SGNN_ERR_INVALID_ARGUMENT, "%s: bad size", who);
    SGNN_REQUIRE(n < (1LL << 31) && C < (1LL << 31) && K <= 16384, SGNN_ERR_TOO_LARGE, "%s: too large", who);
    return SGNN_OK;
}

struct NllCall {
    const void *x;
    int64_t ldx;
    const void *w;
    int64_t ldw;
    NllBias bias;
    const int64_t *labels;
    const uint8_t *mask;
    float inv_count;
    int64_t n, K, C;
    float *loss, *lse;
    void *gx;
    int64_t ldgx;
    void *gw;
    int64_t ldgw;
    void *gb;
    char *ws;
    cudaStream_t s;
};

template <class T>
static int nll_run(const NllCall &c)
{
    const bool grad = c.gx != nullptr;
    const NllSizes z = nll_sizes(c.n, c.K, c.C, grad);
    int *counts = reinterpret_cast<int *>(c.ws + z.counts), *rows = reinterpret_cast<int *>(c.ws + z.rows);
    int *total = reinterpret_cast<int *>(c.ws + z.total);
    float2 *run = reinterpret_cast<float2 *>(c.ws + z.run);
    float *picked = reinterpret_cast<float *>(c.ws + z.picked), *lse = reinterpret_cast<float *>(c.ws + z.lse);
    float *acc = reinterpret_cast<float *>(c.ws + z.acc), *piece = reinterpret_cast<float *>(c.ws + z.piece);
    cudaStream_t s = c.s;
    nll_count_kernel<<<(unsigned)z.blocks, kListThreads, 0, s>>>(c.labels, c.mask, c.n, c.C, counts);
    nll_list_kernel<<<(unsigned)z.blocks, kListThreads, 0, s>>>(c.labels, c.mask, c.n, c.C, counts, rows, total);
    if (c.lse) SGNN_CUDA_OK(cudaMemsetAsync(c.lse, 0, c.n * 4, s));
    const RowsOperand<T> xa{static_cast<const T *>(c.x), c.ldx, rows, total, (int)c.K};
    const auto logits = [&](int64_t first, int64_t width) {
        const WeightOperand<T> wb{static_cast<const T *>(c.w), c.ldw, first, c.C, (int)c.K};
        const dim3 grid((unsigned)ceil_div(width, kTile), (unsigned)ceil_div(c.n, kTile), 1);
        tile_product_kernel<<<grid, kTileThreads, 0, s>>>(xa, wb, PieceStore{piece, width, total}, c.K, c.K);
        return wb;
    };
    for (int64_t first = 0; first < c.C; first += z.width) {
        const int64_t width = c.C - first < z.width ? c.C - first : z.width;
        logits(first, width);
        nll_stats_kernel<T><<<(unsigned)c.n, 256, 0, s>>>(piece, first, width, c.bias, c.labels, rows, total, run, picked);
    }
    nll_lse_kernel<<<(unsigned)ceil_div(c.n, 256), 256, 0, s>>>(run, rows, total, lse, c.lse);
    nll_loss_kernel<<<1, 1024, 0, s>>>(lse, picked, total, c.inv_count, c.loss);
    SGNN_LAUNCH_OK("linear_nll_loss");
    if (!grad) return SGNN_OK;
    SGNN_CUDA_OK(cudaMemsetAsync(acc, 0, c.n * c.K * 4, s));
    for (int64_t first = 0; first < c.C; first += z.width) {
        const int64_t width = c.C - first < z.width ? c.C - first : z.width;
        const WeightOperand<T> wb = logits(first, width);
        nll_piece_grad_kernel<T><<<(unsigned)c.n, 256, 0, s>>>(piece, first, width, c.bias, c.labels, rows, total, lse);
        const PieceOperand g{piece, width, total};
        const dim3 grid_x((unsigned)ceil_div(c.K, kTile), (unsigned)ceil_div(c.n, kTile), 1);
        tile_product_kernel<<<grid_x, kTileThreads, 0, s>>>(g, WeightOperandT<T>{wb}, AddRows{acc, (int)c.K, total}, width, width);
        const dim3 grid_w((unsigned)ceil_div(c.K, kTile), (unsigned)ceil_div(width, kTile), 1);
        tile_product_kernel<<<grid_w, kTileThreads, 0, s>>>(
            PieceOperandT{g}, RowsOperandT<T>{xa}, WeightStore<T>{static_cast<T *>(c.gw), c.ldgw, first, width, (int)c.K, c.inv_count},
            c.n, c.n);
        if (c.gb)
            nll_bias_grad_kernel<T><<<(unsigned)ceil_div(width, 128), 128, 0, s>>>(piece, first, width, total, c.inv_count, c.bias.f32, c.gb);
    }
    SGNN_CUDA_OK(cudaMemset2DAsync(c.gx, c.ldgx * sizeof(T), 0, c.K * sizeof(T), c.n, s));
    nll_rows_out_kernel<T><<<(unsigned)c.n, 128, 0, s>>>(acc, rows, total, c.inv_count, static_cast<T *>(c.gx), c.ldgx, (int)c.K);
    SGNN_LAUNCH_OK("linear_nll_loss gradient");
    return SGNN_OK;
}

}  // namespace sgnn

using namespace sgnn;

extern "C" SGNN_API int sgnn_linear_nll_workspace_bytes(int dtype, int64_t n, int64_t K, int64_t C, int with_grad, size_t *bytes)
{
    const char *who = "linear_nll_workspace_bytes";
    int rc = nll_check(who, dtype, n, K, C);
    if (rc) return rc;
    SGNN_REQUIRE(bytes != nullptr, SGNN_ERR_INVALID_ARGUMENT, "%s: null result pointer", who);
    *bytes = n == 0 ? 0 : nll_sizes(n, K, C, with_grad != 0).bytes;
    return SGNN_OK;
}

extern "C" SGNN_API int sgnn_linear_nll_loss(int dtype, const void *d_x, int64_t ldx, const void *d_w, int64_t ldw,
                                             int bias_dtype, const void *d_bias, const int64_t *d_labels,
                                             const uint8_t *d_mask, float inv_count, int64_t n, int64_t K, int64_t C,
                                             float *d_loss, float *d_lse, void *d_gx, int64_t ldgx, void *d_gw,
                                             int64_t ldgw, void *d_gb, void *d_workspace, size_t workspace_bytes, void *stream)
{
    const char *who = "linear_nll_loss";
    int rc = nll_check(who, dtype, n, K, C);
    if (rc) return rc;
    SGNN_REQUIRE(bias_dtype == SGNN_F32 || bias_dtype == dtype, SGNN_ERR_INVALID_ARGUMENT,
                 "%s: the bias must be fp32 or of the type of x", who);
    SGNN_REQUIRE(inv_count == inv_count, SGNN_ERR_INVALID_ARGUMENT, "%s: inv_count is NaN", who);
    SGNN_REQUIRE(d_loss != nullptr, SGNN_ERR_INVALID_ARGUMENT, "%s: null output", who);
    SGNN_REQUIRE((n == 0 || (d_gx == nullptr) == (d_gw == nullptr)) && (d_gb == nullptr || (d_gw != nullptr && d_bias != nullptr)),
                 SGNN_ERR_INVALID_ARGUMENT, "%s: gx and gw belong together, gb needs them and a bias", who);
    const size_t b = elem_bytes(dtype);
    cudaStream_t s = (cudaStream_t)stream;
    SGNN_REQUIRE(d_gw == nullptr || (ldgw >= K && ldgx >= K), SGNN_ERR_INVALID_ARGUMENT,
                 "%s: leading dimension shorter than a row", who);
    if (n == 0) {
        SGNN_CUDA_OK(cudaMemsetAsync(d_loss, 0, sizeof(float), s));
        if (d_gw) SGNN_CUDA_OK(cudaMemset2DAsync(d_gw, ldgw * b, 0, K * b, C, s));
        if (d_gb) SGNN_CUDA_OK(cudaMemsetAsync(d_gb, 0, C * elem_bytes(bias_dtype), s));
        return SGNN_OK;
    }
    SGNN_REQUIRE(d_x && d_w && d_labels, SGNN_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
    SGNN_REQUIRE((n == 1 || ldx >= K) && (C == 1 || ldw >= K), SGNN_ERR_INVALID_ARGUMENT, "%s: leading dimension shorter than a row", who);
    size_t need = 0;
    rc = sgnn_linear_nll_workspace_bytes(dtype, n, K, C, d_gx != nullptr, &need);
    if (rc) return rc;
    SGNN_REQUIRE(d_workspace != nullptr && workspace_bytes >= need && reinterpret_cast<uintptr_t>(d_workspace) % 256 == 0,
                 SGNN_ERR_WORKSPACE, "%s: 256-byte aligned workspace of %zu bytes needed, %zu given", who, need, workspace_bytes);
    const NllCall c{d_x, ldx, d_w, ldw, NllBias{d_bias, bias_dtype == SGNN_F32}, d_labels, d_mask, inv_count, n, K, C, d_loss,
                    d_lse, d_gx, ldgx, d_gw, ldgw, d_gb, static_cast<char *>(d_workspace), s};
    return dtype == SGNN_F32 ? nll_run<float>(c) : nll_run<__nv_bfloat16>(c);
}
