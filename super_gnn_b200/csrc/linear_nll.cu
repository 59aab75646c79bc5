// Negative log-likelihood of a linear classifier over many classes and its gradients (sm_100a), in pieces of the
// classes, so that the logits z = x W^T + b, [n, C], are never kept:
//
//     lse[r] = log sum_c exp z[r, c]        running maximum and sum over the pieces
//     loss   = inv_count sum_r (lse[r] - z[r, label])
//     G      = inv_count (exp(z - lse) - onehot)  piece by piece, from logits computed a second time
//     gx += G W_piece,  gw_piece = G^T x,  gb_piece = sum_r G
//
// The rows in the loss are listed first (in order) and copied together, so that a row outside the mask costs nothing and
// whatever it holds is not read.  The products run on the tensor cores (nll_product.cuh): 8 m C K operations for m rows,
// of which 2 m C K compute the logits again, the price of not keeping them.  Rows go in chunks of up to 32768, classes in
// pieces, so that G (16 bits an element, rows of the chunk x classes of the piece) stays in the L2 cache between the
// kernel that writes it and the two products that read it.
//
// bf16 operands enter the products as they are; G is rounded to bf16, as it is between two bf16 layers.  fp32 operands are
// split into two fp16 planes, v 2^e = v0 + v1 with 2^e bringing the largest value of the row below 2^15: 22 bits of every
// value that is not 2^-16 of the largest, an absolute 2^-39 of the largest below that.  A product of two such operands
// takes three products of planes (v1 w1 is below 2^-22).  The scale belongs to a row for the logits, where rows of x meet
// rows of W, and to a column for the gradients, where columns come out: two sets of planes of each.  bf16 terms would need
// no scale but six products for the same accuracy.
#include "nll_product.cuh"
#include "row_io.cuh"

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


struct NllBias {
    const void *b;
    bool f32;
};
template <class T>
__device__ __forceinline__ float bias_at(NllBias b, int64_t c)
{
    return b.b == nullptr ? 0.f : b.f32 ? static_cast<const float *>(b.b)[c] : to_f32<T>(static_cast<const T *>(b.b)[c]);
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// bias log2(e) of the classes, -inf up to the end of the last tile: classes that are not there have probability 0 (their
// rows of W read as zeros, scaled by 1)
template <class T>
__global__ void nll_bias_kernel(NllBias bias, int64_t C, int64_t padded, float *__restrict__ bias2, float *__restrict__ w_down,
                                int *__restrict__ failed)
{
    const int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (c == 0) *failed = 0;
    if (c < padded) bias2[c] = c < C ? bias_at<T>(bias, c) * kLog2e : -INFINITY;
    if (c >= C && c < padded && w_down != nullptr) w_down[c] = 1.0f;
}

// 2^e that brings `largest` into [2^14, 2^15), and 2^-e; 1 for nothing but zeros and for what is not finite
__device__ __forceinline__ void plane_scale(float largest, float &up, float &down)
{
    up = down = 1.0f;
    if (!(largest > 0.f) || !(largest <= FLT_MAX)) return;
    int e = 14 - ((int)(__float_as_uint(largest) >> 23) - 127);
    e = e < -126 ? -126 : e > 126 ? 126 : e;
    up = __uint_as_float((unsigned)(e + 127) << 23);
    down = __uint_as_float((unsigned)(127 - e) << 23);
}

// Where the rows of a matrix come from: row i is src[rows[i]] for i < *total, or src[i] for i < count
struct RowSource {
    const void *src;
    int64_t ld;
    const int *rows, *total;
    int64_t count;
    int K;
};
__device__ __forceinline__ int64_t source_rows(const RowSource &s) { return s.total ? *s.total : s.count; }
__device__ __forceinline__ int64_t source_row(const RowSource &s, int64_t i) { return s.rows ? s.rows[i] : i; }

// Planes of a matrix, [1 or 2][rows][ld] 16-bit, zero in columns K .. ld
struct Planes {
    uint16_t *p;
    int64_t ld, stride;
};

// The label's logit of the listed rows, in units of log2, from the operands as they are given
struct Picked {
    const int64_t *labels;
    const void *w;
    int64_t ldw;
    NllBias bias;
    int *label;
    float *picked2;
};

__device__ __forceinline__ void store_split(const Planes &pl, int64_t at, float v, float up)
{
    const float s = v * up;
    const __half h = __float2half_rn(s);
    reinterpret_cast<__half *>(pl.p)[at] = h;
    reinterpret_cast<__half *>(pl.p)[at + pl.stride] = __float2half_rn(s - __half2float(h));
}

// largest |value| of every column, as bits (a NaN or an infinity stays above every number)
__global__ void __launch_bounds__(256) nll_column_max_kernel(RowSource s, unsigned *__restrict__ largest)
{
    __shared__ unsigned part[8][32];
    const int k = blockIdx.x * 32 + (threadIdx.x & 31), g = threadIdx.x >> 5;
    const int64_t n = source_rows(s);
    unsigned m = 0;
    if (k < s.K) {
        for (int64_t i = (int64_t)blockIdx.y * 8 + g; i < n; i += (int64_t)gridDim.y * 8) {
            const unsigned b = __float_as_uint(static_cast<const float *>(s.src)[source_row(s, i) * s.ld + k]) & 0x7fffffffu;
            m = b > m ? b : m;
        }
    }
    part[g][threadIdx.x & 31] = m;
    __syncthreads();
    if (g == 0 && k < s.K) {
        for (int w = 1; w < 8; ++w) m = part[w][threadIdx.x] > m ? part[w][threadIdx.x] : m;
        atomicMax(largest + k, m);
    }
}

__global__ void nll_column_scale_kernel(const unsigned *__restrict__ largest, int K, float *__restrict__ up, float *__restrict__ down)
{
    const int k = blockIdx.x * blockDim.x + threadIdx.x;
    if (k < K) plane_scale(__uint_as_float(largest[k]), up[k], down[k]);
}

// Rows together, one warp a row, and zero rows up to a whole tile behind the listed ones.  fp32 (SPLIT): planes scaled by
// row and, where col.p is given, planes scaled by column.
template <class T, bool SPLIT>
__global__ void __launch_bounds__(256)
nll_take_kernel(RowSource s, Planes row, Planes col, const float *__restrict__ col_up, float *__restrict__ row_down, Picked pick)
{
    const int lane = threadIdx.x & 31;
    const int64_t n = source_rows(s), end = s.total ? (n + kPM - 1) / kPM * kPM : n;
    for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < end; i += (int64_t)gridDim.x * 8) {
        const bool there = i < n;
        const int64_t r = there ? source_row(s, i) : 0;
        const T *x = static_cast<const T *>(s.src) + r * s.ld;
        if (pick.label != nullptr && there) {
            const int64_t label = pick.labels[r];
            const T *w = static_cast<const T *>(pick.w) + label * pick.ldw;
            float z = 0.f;
            for (int k = lane; k < s.K; k += 32) z = __fmaf_rn(to_f32<T>(x[k]), to_f32<T>(w[k]), z);
            z = all_sum(z);
            if (lane == 0) {
                pick.label[i] = (int)label;
                pick.picked2[i] = (z + bias_at<T>(pick.bias, label)) * kLog2e;
            }
        }
        float up = 1.f, down = 1.f;
        if (SPLIT) {
            float largest = 0.f, poison = 0.f;
            for (int k = lane; there && k < s.K; k += 32) {
                const float v = to_f32<T>(x[k]);
                largest = fmaxf(largest, fabsf(v));
                poison = __fmaf_rn(v, 0.f, poison);
            }
            largest = warp_max(largest);
            if (all_sum(poison) == 0.f) plane_scale(largest, up, down);
            if (lane == 0) row_down[i] = down;
        }
        for (int k = lane; k < row.ld; k += 32) {
            const bool in = there && k < s.K;
            const int64_t at = i * row.ld + k;
            if (SPLIT) {
                const float v = in ? to_f32<T>(x[k]) : 0.f;
                store_split(row, at, v, up);
                if (col.p) store_split(col, at, v, k < s.K ? __ldg(col_up + k) : 1.f);
            } else {
                row.p[at] = in ? reinterpret_cast<const uint16_t *>(x)[k] : (uint16_t)0;
            }
        }
    }
}

// lse of the rows of a chunk from the parts of their tiles, and the sum of their losses a block
__global__ void __launch_bounds__(256)
nll_join_kernel(const float2 *__restrict__ stats, int parts, int row0, int row_cap, const int *__restrict__ rows,
                const int *__restrict__ total, const float *__restrict__ picked2, float *__restrict__ lse2,
                float *__restrict__ lse_out, float *__restrict__ loss_part)
{
    __shared__ float2 red[8][32];
    const int lane = threadIdx.x & 31, g = threadIdx.x >> 5;
    const int i = blockIdx.x * 32 + lane;  // of the chunk
    const bool on = i < row_cap && row0 + i < *total;
    float mx = -INFINITY, sum = 0.f;
    if (on) {
        for (int p = g; p < parts; p += 8) {
            const float2 v = stats[(int64_t)p * row_cap + i];
            const float top = fmaxf(mx, v.x), ref = top == -INFINITY ? 0.f : top;
            sum = sum * exp2f(mx - ref) + v.y * exp2f(v.x - ref);
            mx = top;
        }
    }
    red[g][lane] = make_float2(mx, sum);
    __syncthreads();
    if (g != 0) return;
    for (int w = 1; w < 8; ++w) {
        const float2 v = red[w][lane];
        const float top = fmaxf(mx, v.x), ref = top == -INFINITY ? 0.f : top;
        sum = sum * exp2f(mx - ref) + v.y * exp2f(v.x - ref);
        mx = top;
    }
    float loss = 0.f;
    if (on) {
        const float l = mx + log2f(sum);
        lse2[i] = l;
        if (lse_out) lse_out[rows[row0 + i]] = l * kLn2;
        loss = (l - picked2[i]) * kLn2;
    }
    loss = all_sum(loss);
    if (lane == 0) loss_part[blockIdx.x] = loss;
}

__global__ void __launch_bounds__(1024)
nll_loss_kernel(const float *__restrict__ parts, int count, float inv_count, const int *__restrict__ failed, float *__restrict__ loss)
{
    __shared__ float red[32];
    float s = 0.f;
    for (int i = threadIdx.x; i < count; i += 1024) s += parts[i];
    s = all_sum(s);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x < 32) {
        s = all_sum(red[threadIdx.x]);
        if (threadIdx.x == 0) *loss = *failed ? __int_as_float(0x7fffffff) : s * inv_count;
    }
}

// gx of the listed rows of a chunk: the partial sums of the splits, scaled back; NaN when a wait gave up before
template <class T>
__global__ void __launch_bounds__(256)
nll_rows_out_kernel(const float *__restrict__ acc, int64_t acc_ld, int64_t acc_split, int splits, int row0, int row_cap,
                    const int *__restrict__ rows, const int *__restrict__ total, float scale, const float *__restrict__ col_down,
                    const int *__restrict__ failed, T *__restrict__ gx, int64_t ldgx, int K, float *__restrict__ loss)
{
    const int lane = threadIdx.x & 31;
    const bool bad = *failed != 0;
    if (bad && blockIdx.x == 0 && threadIdx.x == 0) *loss = __int_as_float(0x7fffffff);
    for (int i = blockIdx.x * 8 + (threadIdx.x >> 5); i < row_cap && row0 + i < *total; i += gridDim.x * 8) {
        T *out = gx + (int64_t)rows[row0 + i] * ldgx;
        for (int k = lane; k < K; k += 32) {
            float v = 0.f;
            for (int s = 0; s < splits; ++s) v += acc[s * acc_split + (int64_t)i * acc_ld + k];
            v *= scale;
            if (col_down) v *= col_down[k];
            out[k] = from_f32<T>(bad ? __int_as_float(0x7fffffff) : v);
        }
    }
}

// gw and gb from the partial sums of the splits (and of all chunks)
template <class T>
__global__ void __launch_bounds__(256)
nll_weight_out_kernel(const float *__restrict__ acc, int64_t acc_ld, int64_t acc_split, const float *__restrict__ bias_acc,
                      int64_t bias_split, int splits, int64_t C, int K, float scale, const float *__restrict__ col_down,
                      T *__restrict__ gw, int64_t ldgw, bool gb_f32, void *__restrict__ gb)
{
    const int lane = threadIdx.x & 31;
    for (int64_t c = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); c < C; c += (int64_t)gridDim.x * 8) {
        for (int k = lane; k < K; k += 32) {
            float v = 0.f;
            for (int s = 0; s < splits; ++s) v += acc[s * acc_split + c * acc_ld + k];
            v *= scale;
            if (col_down) v *= col_down[k];
            gw[c * ldgw + k] = from_f32<T>(v);
        }
        if (lane == 0 && gb != nullptr) {
            float v = 0.f;
            for (int s = 0; s < splits; ++s) v += bias_acc[s * bias_split + c];
            if (gb_f32) static_cast<float *>(gb)[c] = v * scale;
            else static_cast<T *>(gb)[c] = from_f32<T>(v * scale);
        }
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
constexpr int64_t kNllRowCap = 32768;             // rows of a chunk
constexpr int64_t kNllPieceBytes = 64ll << 20;    // of G: half of the L2 cache

static int64_t round_up(int64_t v, int64_t to) { return ceil_div(v, to) * to; }

// Splits of a reduction of `blocks` steps for `tiles` result tiles: the fewest that keep nine of ten SMs busy (or the
// best there is), each with at least four steps.
static int nll_splits(int64_t tiles, int64_t blocks)
{
    const int64_t sms = sm_count();
    int64_t most = blocks / 4, best = 1;
    if (most > 148) most = 148;
    double best_use = 0;
    for (int64_t s = 1; s <= most; ++s) {
        const int64_t units = tiles * s;
        const double use = (double)units / (double)(round_up(units, sms));
        if (use > best_use + 1e-9) best = s, best_use = use;
        if (use >= 0.9) break;
    }
    return (int)best;
}

struct NllPlan {
    int planes;
    int64_t blocks, padded, row_cap, chunks, cls_padded, piece, pieces, ld, acc_ld;
    int row_splits, weight_splits;
    bool copy_w, weights_direct;
    size_t counts, rows, total, failed, label, picked2, lse2, loss_part, bias2, stats;
    size_t x_row, x_col, w_row, w_col, x_down, w_down, x_largest, w_largest, x_up, x_cdown, w_up, w_cdown;
    size_t grad, acc_x, acc_w, bias_acc, bytes;
};

// `copy_w`: bf16 weights whose rows TMA cannot read where they are.  The size query allows for the copy.
static NllPlan nll_plan(int dtype, int64_t n, int64_t K, int64_t C, bool grad, bool copy_w)
{
    NllPlan p{};
    const bool f32 = dtype == SGNN_F32;
    p.planes = f32 ? 2 : 1;
    p.copy_w = f32 || copy_w;
    p.blocks = ceil_div(n, kListRows);
    p.padded = round_up(n, kPM);
    p.row_cap = p.padded < kNllRowCap ? p.padded : kNllRowCap;
    p.chunks = ceil_div(p.padded, p.row_cap);
    p.cls_padded = round_up(C, kPN);
    p.piece = kNllPieceBytes / (2 * p.planes * p.row_cap) / kPN * kPN;
    if (p.piece < kPN) p.piece = kPN;
    if (p.piece > p.cls_padded) p.piece = p.cls_padded;
    p.pieces = ceil_div(p.cls_padded, p.piece);
    p.ld = round_up(K, 8);
    p.acc_ld = round_up(K, 32);
    const int64_t tiles_k = ceil_div(K, kPN);
    p.row_splits = nll_splits(p.row_cap / kPM * tiles_k, p.piece / kPK);
    p.weight_splits = nll_splits(p.piece / kPM * tiles_k, p.row_cap / kPK);
    p.weights_direct = p.chunks == 1 && p.weight_splits == 1;
    size_t at = 0;
    const auto take = [&at](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    const size_t mat_x = (size_t)p.planes * p.padded * p.ld * 2, mat_w = (size_t)p.planes * C * p.ld * 2;
    p.counts = take(p.blocks * 4), p.rows = take(n * 4), p.total = take(4), p.failed = take(4);
    p.label = take(p.padded * 4), p.picked2 = take(p.padded * 4), p.lse2 = take(p.row_cap * 4);
    p.loss_part = take(ceil_div(p.padded, 32) * 4), p.bias2 = take(p.cls_padded * 4);
    p.stats = take((size_t)p.cls_padded / 128 * p.row_cap * 8);
    p.x_row = take(mat_x), p.w_row = take(p.copy_w ? mat_w : 0);
    if (f32) {
        p.x_down = take(p.padded * 4), p.w_down = take(p.cls_padded * 4);
        if (grad) {
            p.x_col = take(mat_x), p.w_col = take(mat_w);
            p.x_largest = take(2 * K * 4), p.w_largest = p.x_largest + K * 4;  // one clear for both
            p.x_up = take(K * 4), p.x_cdown = take(K * 4), p.w_up = take(K * 4), p.w_cdown = take(K * 4);
        }
    }
    if (grad) {
        p.grad = take((size_t)p.planes * p.row_cap * p.piece * 2);
        p.acc_x = take((size_t)p.row_splits * p.row_cap * p.acc_ld * 4);
        p.acc_w = take(p.weights_direct ? 0 : (size_t)p.weight_splits * C * p.acc_ld * 4);
        p.bias_acc = take(p.weights_direct ? 0 : (size_t)p.weight_splits * C * 4);
    }
    p.bytes = at;
    return p;
}

struct NllCall {
    int dtype;
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

static bool nll_must_copy_weights(int dtype, const void *w, int64_t ldw, int64_t C)
{
    return dtype == SGNN_BF16 && !(aligned16(w) && ldw % 8 == 0 && C > 1);
}

template <int KIND, int PLANES>
static int nll_product(const ProductCall &c, int64_t units, cudaStream_t s)
{
    constexpr int smem = ProductShared<PLANES>::kBytes;
    SGNN_CUDA_OK(cudaFuncSetAttribute(nll_product_kernel<KIND, PLANES>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    const int64_t grid = units < sm_count() ? units : sm_count();
    nll_product_kernel<KIND, PLANES><<<(unsigned)grid, kPThreads, smem, s>>>(c);
    SGNN_LAUNCH_OK("linear_nll product");
    return SGNN_OK;
}

template <class T, int PLANES>
static int nll_run(const NllCall &c)
{
    constexpr bool f32 = PLANES == 2;
    const bool grad = c.gx != nullptr;
    const NllPlan p = nll_plan(c.dtype, c.n, c.K, c.C, grad, nll_must_copy_weights(c.dtype, c.w, c.ldw, c.C));
    const auto ints = [&](size_t at) { return reinterpret_cast<int *>(c.ws + at); };
    const auto floats = [&](size_t at) { return reinterpret_cast<float *>(c.ws + at); };
    const auto halves = [&](size_t at) { return reinterpret_cast<uint16_t *>(c.ws + at); };
    cudaStream_t s = c.s;
    int rc;

    // the rows in the loss
    if (p.blocks > 1)
        nll_count_kernel<<<(unsigned)p.blocks, kListThreads, 0, s>>>(c.labels, c.mask, c.n, c.C, ints(p.counts));
    nll_list_kernel<<<(unsigned)p.blocks, kListThreads, 0, s>>>(c.labels, c.mask, c.n, c.C, ints(p.counts), ints(p.rows), ints(p.total));
    nll_bias_kernel<T><<<(unsigned)ceil_div(p.cls_padded, 256), 256, 0, s>>>(c.bias, c.C, p.cls_padded, floats(p.bias2),
                                                                              f32 ? floats(p.w_down) : nullptr, ints(p.failed));
    if (c.lse) SGNN_CUDA_OK(cudaMemsetAsync(c.lse, 0, c.n * 4, s));
    if (grad) SGNN_CUDA_OK(cudaMemset2DAsync(c.gx, c.ldgx * sizeof(T), 0, c.K * sizeof(T), c.n, s));

    // the operands as the products read them
    const RowSource xs{c.x, c.ldx, ints(p.rows), ints(p.total), 0, (int)c.K}, wsrc{c.w, c.ldw, nullptr, nullptr, c.C, (int)c.K};
    const Planes x_row{halves(p.x_row), p.ld, p.padded * p.ld}, w_row{halves(p.w_row), p.ld, c.C * p.ld};
    const bool cols = f32 && grad;
    const Planes x_col{cols ? halves(p.x_col) : nullptr, p.ld, p.padded * p.ld}, w_col{cols ? halves(p.w_col) : nullptr, p.ld, c.C * p.ld};
    if (cols) {
        SGNN_CUDA_OK(cudaMemsetAsync(c.ws + p.x_largest, 0, 2 * c.K * 4, s));
        const int64_t tall = 4 * sm_count();
        const dim3 gx((unsigned)ceil_div(c.K, 32), (unsigned)(ceil_div(c.n, 64) < tall ? ceil_div(c.n, 64) : tall));
        const dim3 gw((unsigned)ceil_div(c.K, 32), (unsigned)(ceil_div(c.C, 64) < tall ? ceil_div(c.C, 64) : tall));
        unsigned *xl = reinterpret_cast<unsigned *>(c.ws + p.x_largest), *wl = reinterpret_cast<unsigned *>(c.ws + p.w_largest);
        nll_column_max_kernel<<<gx, 256, 0, s>>>(xs, xl);
        nll_column_max_kernel<<<gw, 256, 0, s>>>(wsrc, wl);
        nll_column_scale_kernel<<<(unsigned)ceil_div(c.K, 256), 256, 0, s>>>(xl, (int)c.K, floats(p.x_up), floats(p.x_cdown));
        nll_column_scale_kernel<<<(unsigned)ceil_div(c.K, 256), 256, 0, s>>>(wl, (int)c.K, floats(p.w_up), floats(p.w_cdown));
    }
    const int64_t wide = 16 * sm_count();
    const Picked pick{c.labels, c.w, c.ldw, c.bias, ints(p.label), floats(p.picked2)};
    nll_take_kernel<T, f32><<<(unsigned)(p.padded / 8 < wide ? p.padded / 8 : wide), 256, 0, s>>>(
        xs, x_row, x_col, cols ? floats(p.x_up) : nullptr, f32 ? floats(p.x_down) : nullptr, pick);
    if (p.copy_w)
        nll_take_kernel<T, f32><<<(unsigned)(ceil_div(c.C, 8) < wide ? ceil_div(c.C, 8) : wide), 256, 0, s>>>(
            wsrc, w_row, w_col, cols ? floats(p.w_up) : nullptr, f32 ? floats(p.w_down) : nullptr, Picked{});
    SGNN_LAUNCH_OK("linear_nll operands");

    // tensor maps: x and W along k (rows of a tile at once) and across it (64 steps of the reduction at once), G likewise
    ProductCall lc{}, rc_{}, wc{};
    const void *wp = p.copy_w ? (const void *)w_row.p : c.w;
    const int64_t wld = p.copy_w ? p.ld : c.ldw, wst = p.copy_w ? w_row.stride : c.C * c.ldw;
    if ((rc = umma_tensor_map(&lc.a, x_row.p, !f32, c.K, p.padded, p.ld, PLANES, x_row.stride, kPM))) return rc;
    if ((rc = umma_tensor_map(&lc.b, wp, !f32, c.K, c.C, wld, PLANES, wst, kPN))) return rc;
    lc.total = ints(p.total), lc.failed = ints(p.failed), lc.feats = (int)c.K, lc.splits = 1, lc.bf16 = !f32;
    lc.bias2 = floats(p.bias2), lc.row_scale = f32 ? floats(p.x_down) : nullptr, lc.cls_scale = f32 ? floats(p.w_down) : nullptr;
    lc.stats = reinterpret_cast<float2 *>(c.ws + p.stats), lc.row_cap = (int)p.row_cap, lc.lse2 = floats(p.lse2);
    lc.scale = c.inv_count * (f32 ? 1.0f / kGradScale : 1.0f);
    if (grad) {
        lc.grad = halves(p.grad), lc.grad_ld = p.piece;
        rc_ = lc, wc = lc;
        const int64_t plane = p.row_cap * p.piece;
        if ((rc = umma_tensor_map(&rc_.a, lc.grad, !f32, p.piece, p.row_cap, p.piece, PLANES, plane, kPM))) return rc;
        if ((rc = umma_tensor_map(&rc_.b, f32 ? (const void *)w_col.p : wp, !f32, c.K, c.C, wld, PLANES, wst, kPK))) return rc;
        if ((rc = umma_tensor_map(&wc.a, lc.grad, !f32, p.piece, p.row_cap, p.piece, PLANES, plane, kPK))) return rc;
        if ((rc = umma_tensor_map(&wc.b, f32 ? x_col.p : x_row.p, !f32, c.K, p.padded, p.ld, PLANES, x_row.stride, kPK))) return rc;
        rc_.splits = p.row_splits, rc_.out = floats(p.acc_x), rc_.out_ld = p.acc_ld, rc_.out_split = p.row_cap * p.acc_ld;
        wc.splits = p.weight_splits, wc.out_ld = p.acc_ld, wc.out_split = c.C * p.acc_ld, wc.bias_split = c.C;
        wc.col_scale = f32 ? floats(p.x_cdown) : nullptr;
        if (p.weights_direct)
            wc.gw = c.gw, wc.gw_ld = c.ldgw, wc.gb = c.gb, wc.gw_f32 = f32, wc.gb_f32 = c.bias.f32;
    }
    const int64_t tiles_k = ceil_div(c.K, kPN), loss_blocks = ceil_div(p.row_cap, 32);
    for (int64_t q = 0; q < p.chunks; ++q) {
        const int row0 = (int)(q * p.row_cap);
        for (ProductCall *k : {&lc, &rc_, &wc}) k->row0 = row0;
        lc.label = ints(p.label) + row0, lc.picked2 = floats(p.picked2) + row0;
        lc.cls0 = 0, lc.cls_count = (int)c.C;
        const int64_t tiles_m = p.row_cap / kPM;
        if ((rc = nll_product<kLogitStats, PLANES>(lc, tiles_m * ceil_div(c.C, kPN), s))) return rc;
        const int64_t left = p.padded - row0 < p.row_cap ? p.padded - row0 : p.row_cap;
        nll_join_kernel<<<(unsigned)ceil_div(left, 32), 256, 0, s>>>(lc.stats, (int)(p.cls_padded / 128), row0, (int)p.row_cap,
                                                                     ints(p.rows), ints(p.total), lc.picked2, floats(p.lse2), c.lse,
                                                                     floats(p.loss_part) + q * loss_blocks);
        SGNN_LAUNCH_OK("linear_nll join");
        if (!grad) continue;
        for (int64_t first = 0; first < c.C; first += p.piece) {
            const int64_t count = c.C - first < p.piece ? c.C - first : p.piece;
            for (ProductCall *k : {&lc, &rc_, &wc}) k->cls0 = (int)first, k->cls_count = (int)count;
            if ((rc = nll_product<kLogitGrad, PLANES>(lc, tiles_m * ceil_div(count, kPN), s))) return rc;
            rc_.add = first > 0;
            if ((rc = nll_product<kRowGrad, PLANES>(rc_, tiles_m * tiles_k * p.row_splits, s))) return rc;
            wc.add = q > 0;
            if (!p.weights_direct) wc.out = floats(p.acc_w) + first * p.acc_ld, wc.bias_out = floats(p.bias_acc) + first;
            if ((rc = nll_product<kWeightGrad, PLANES>(wc, ceil_div(count, kPM) * tiles_k * p.weight_splits, s))) return rc;
        }
        if (q + 1 < p.chunks) {
            nll_rows_out_kernel<T><<<(unsigned)(left / 8 < wide ? left / 8 : wide), 256, 0, s>>>(
                floats(p.acc_x), p.acc_ld, rc_.out_split, p.row_splits, row0, (int)p.row_cap, ints(p.rows), ints(p.total), lc.scale,
                f32 ? floats(p.w_cdown) : nullptr, ints(p.failed), static_cast<T *>(c.gx), c.ldgx, (int)c.K, c.loss);
        }
    }
    nll_loss_kernel<<<1, 1024, 0, s>>>(floats(p.loss_part), (int)ceil_div(p.padded, 32), c.inv_count, ints(p.failed), c.loss);
    if (grad) {
        const int row0 = (int)((p.chunks - 1) * p.row_cap);
        const int64_t left = p.padded - row0;
        nll_rows_out_kernel<T><<<(unsigned)(left / 8 < wide ? left / 8 : wide), 256, 0, s>>>(
            floats(p.acc_x), p.acc_ld, rc_.out_split, p.row_splits, row0, (int)p.row_cap, ints(p.rows), ints(p.total), lc.scale,
            f32 ? floats(p.w_cdown) : nullptr, ints(p.failed), static_cast<T *>(c.gx), c.ldgx, (int)c.K, c.loss);
        if (!p.weights_direct)
            nll_weight_out_kernel<T><<<(unsigned)(ceil_div(c.C, 8) < wide ? ceil_div(c.C, 8) : wide), 256, 0, s>>>(
                floats(p.acc_w), p.acc_ld, wc.out_split, floats(p.bias_acc), wc.bias_split, p.weight_splits, c.C, (int)c.K, lc.scale,
                f32 ? floats(p.x_cdown) : nullptr, static_cast<T *>(c.gw), c.ldgw, c.bias.f32, c.gb);
    }
    SGNN_LAUNCH_OK("linear_nll_loss");
    return SGNN_OK;
}

static int nll_check(const char *who, int dtype, int64_t n, int64_t K, int64_t C)
{
    SGNN_REQUIRE(dtype == SGNN_F32 || dtype == SGNN_BF16, SGNN_ERR_INVALID_ARGUMENT, "%s: fp32 or bf16 only", who);
    SGNN_REQUIRE(n >= 0 && K > 0 && C > 0, SGNN_ERR_INVALID_ARGUMENT, "%s: bad size", who);
    SGNN_REQUIRE(n <= (1LL << 30) && C <= (1LL << 30) && K <= 16384, SGNN_ERR_TOO_LARGE, "%s: too large", who);
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
    *bytes = n == 0 ? 0 : nll_plan(dtype, n, K, C, with_grad != 0, true).bytes;
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
    const NllCall c{dtype, d_x, ldx, d_w, ldw, NllBias{d_bias, bias_dtype == SGNN_F32}, d_labels, d_mask, inv_count, n, K, C, d_loss,
                    d_lse, d_gx, ldgx, d_gw, ldgw, d_gb, static_cast<char *>(d_workspace), s};
    return dtype == SGNN_F32 ? nll_run<float, 2>(c) : nll_run<__nv_bfloat16, 1>(c);
}
