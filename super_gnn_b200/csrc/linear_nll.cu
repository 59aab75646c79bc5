// Negative log-likelihood of a linear classifier over many classes and its gradients (sm_100a), in pieces of the
// classes, so that the logits z = x W^T + b, [n, C], are never kept:
//
//     lse[r] = log sum_c exp z[r, c]        maximum and sum of every 128 classes, joined in a tree
//     loss   = inv_count sum_r (lse[r] - z[r, label])   both from the same sums: a row that is certain of its label adds 0
//     G      = inv_count (exp(z - lse) - onehot)  piece by piece, from logits computed a second time
//     gx += G W_piece,  gw_piece = G^T x,  gb_piece = sum_r G
//
// The rows in the loss are listed first (in order) and copied together, so that a row outside the mask costs nothing and
// whatever it holds is not read.  The products run on the tensor cores (nll_product.cuh): 8 m C K operations for m rows,
// of which 2 m C K compute the logits again, the price of not keeping them.  Rows go in chunks and classes in pieces,
// and only G of one chunk and one piece exists at a time, 16 bits an element.
//
// bf16 operands enter the products as they are; G is rounded to bf16, as it is between two bf16 layers.  fp32 operands are
// split into two fp16 planes, v 2^e = v0 + v1 with 2^e bringing the largest value of the row below 2^15: 22 bits of every
// value that is not below 2^-16 of the largest, an absolute 2^-39 of the largest below that (in the gradients 2^-27 and 2^-50, see
// kSecondPlane).  A product of two such operands takes three products of planes (v1 w1 is below 2^-22).  The scale belongs to a row
// for the logits, where rows of x meet rows of W, and to a column for the gradients, where columns come out: two sets of
// planes of each.  bf16 terms would need no scale but six products for the same accuracy.
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
    __shared__ int part[kListThreads / 32];
    let_next_kernel_start();
    wait_for_kernels_before();
    int c = 0;
#pragma unroll
    for (int i = 0; i < kListRows / kListThreads; ++i)
        c += in_loss(labels, mask, (int64_t)blockIdx.x * kListRows + i * kListThreads + threadIdx.x, n, C) ? 1 : 0;
    c = __reduce_add_sync(FULL, c);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = c;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kListThreads / 32; ++w) c += part[w];
        counts[blockIdx.x] = c;
    }
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

// The first `blocks` blocks list the rows in the loss: rows[0 .. m) ascending, *total = m (`counts`: rows in the loss of
// every listing block before).  The others set what the later kernels start from: bias log2(e) of the classes, -inf up to
// the end of the last tile (classes that are not there have probability 0; their rows of W read as zeros, scaled by 1),
// lse = 0 and gx = 0 of all rows, and the counters.
struct NllStart {
    const int64_t *labels;
    const uint8_t *mask;
    int64_t n, C, padded;  // padded: classes of whole tiles
    const int *counts;
    int *rows, *total;
    int blocks;
    NllBias bias;
    float *bias2, *w_down, *lse;
    int *failed, *joined;
    unsigned *largest;  // 2 K of them, or nullptr
    int K;
    void *gx;
    int64_t ldgx;
};

template <class T>
__global__ void __launch_bounds__(kListThreads) nll_start_kernel(const NllStart a)
{
    let_next_kernel_start();
    wait_for_kernels_before();
    if ((int)blockIdx.x >= a.blocks) {
        const int64_t first = (int64_t)(blockIdx.x - a.blocks) * kListThreads + threadIdx.x;
        const int64_t step = (int64_t)(gridDim.x - a.blocks) * kListThreads;
        if (first == 0) *a.failed = 0, *a.joined = 0;
        for (int64_t c = first; c < a.padded; c += step) {
            a.bias2[c] = c < a.C ? bias_at<T>(a.bias, c) * kLog2e : -INFINITY;
            if (c >= a.C && a.w_down != nullptr) a.w_down[c] = 1.0f;
        }
        if (a.lse != nullptr)
            for (int64_t i = first; i < a.n; i += step) a.lse[i] = 0.f;
        if (a.largest != nullptr)
            for (int64_t k = first; k < 2 * a.K; k += step) a.largest[k] = 0u;
        if (a.gx != nullptr) {
            T *gx = static_cast<T *>(a.gx);
            const int64_t all = a.n * a.K;
            if (a.ldgx == a.K && (reinterpret_cast<uintptr_t>(gx) & 15) == 0) {
                constexpr int64_t per = 16 / sizeof(T);
                for (int64_t i = first; i < all / per; i += step) reinterpret_cast<uint4 *>(gx)[i] = make_uint4(0, 0, 0, 0);
                if (first < all % per) gx[all / per * per + first] = from_f32<T>(0.f);
            } else {
                for (int64_t i = first; i < all; i += step) gx[i / a.K * a.ldgx + i % a.K] = from_f32<T>(0.f);
            }
        }
        return;
    }
    __shared__ int part[kListThreads / 32], before[kListThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int s = 0;
    for (int b = threadIdx.x; b < (int)blockIdx.x; b += kListThreads) s += a.counts[b];
    s = __reduce_add_sync(FULL, s);
    if (lane == 0) part[warp] = s;
    __syncthreads();
    int at = 0;
    for (int w = 0; w < kListThreads / 32; ++w) at += part[w];
    unsigned ons = 0;
#pragma unroll
    for (int i = 0; i < kListRows / kListThreads; ++i)
        ons |= in_loss(a.labels, a.mask, (int64_t)blockIdx.x * kListRows + i * kListThreads + threadIdx.x, a.n, a.C) ? 1u << i : 0u;
    for (int i = 0; i < kListRows / kListThreads; ++i) {
        const int64_t r = (int64_t)blockIdx.x * kListRows + i * kListThreads + threadIdx.x;
        const bool on = (ons >> i & 1u) != 0;
        const unsigned vote = __ballot_sync(FULL, on);
        __syncthreads();
        if (lane == 0) before[warp] = __popc(vote);
        __syncthreads();
        int pos = at + __popc(vote & ((1u << lane) - 1u));
        for (int w = 0; w < kListThreads / 32; ++w) {
            if (w < warp) pos += before[w];
            at += before[w];
        }
        if (on) a.rows[pos] = (int)r;
    }
    if ((int)blockIdx.x == a.blocks - 1 && threadIdx.x == 0) *a.total = at;
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

// The labels of the listed rows
struct Picked {
    const int64_t *labels;
    int *label;
};

// `second`: what the second plane is scaled by beyond the first
__device__ __forceinline__ void store_split(const Planes &pl, int64_t at, float v, float up, float second)
{
    const float s = v * up;
    const __half h = __float2half_rn(s);
    reinterpret_cast<__half *>(pl.p)[at] = h;
    reinterpret_cast<__half *>(pl.p)[at + pl.stride] = __float2half_rn((s - __half2float(h)) * second);
}

// largest |value| of every column of x (z = 0) and W (z = 1), as bits: a NaN or an infinity stays above every number
__global__ void __launch_bounds__(256) nll_column_max_kernel(RowSource x, RowSource w, unsigned *__restrict__ largest)
{
    __shared__ unsigned part[8][32];
    let_next_kernel_start();
    wait_for_kernels_before();
    const RowSource s = blockIdx.z == 0 ? x : w;
    const int k = blockIdx.x * 32 + (threadIdx.x & 31), g = threadIdx.x >> 5;
    const int64_t n = source_rows(s), step = (int64_t)gridDim.y * 8;
    unsigned m = 0;
    if (k < s.K) {
#pragma unroll 4
        for (int64_t i = (int64_t)blockIdx.y * 8 + g; i < n; i += step) {
            const unsigned b = __float_as_uint(static_cast<const float *>(s.src)[source_row(s, i) * s.ld + k]) & 0x7fffffffu;
            m = b > m ? b : m;
        }
    }
    part[g][threadIdx.x & 31] = m;
    __syncthreads();
    if (g == 0 && k < s.K) {
        for (int w8 = 1; w8 < 8; ++w8) m = part[w8][threadIdx.x] > m ? part[w8][threadIdx.x] : m;
        atomicMax(largest + (blockIdx.z == 0 ? 0 : s.K) + k, m);
    }
}

// One side of the operands: where it comes from, its planes scaled by row and (fp32 with gradients) by column
struct TakeSide {
    RowSource src;
    Planes row, col;
    const unsigned *largest;  // of the columns
    float *row_down;
    int blocks;
};

// Rows together, one warp a row, zero rows up to a whole tile behind the listed ones; the first blocks take x, the rest W.
template <class T, bool SPLIT>
__global__ void __launch_bounds__(256) nll_take_kernel(const TakeSide xs, const TakeSide ws, const Picked pick)
{
    let_next_kernel_start();
    wait_for_kernels_before();
    const bool is_x = (int)blockIdx.x < xs.blocks;
    const TakeSide &t = is_x ? xs : ws;
    const RowSource &s = t.src;
    const int lane = threadIdx.x & 31, block = is_x ? blockIdx.x : blockIdx.x - xs.blocks;
    const int64_t n = source_rows(s), end = s.total ? (n + kPM - 1) / kPM * kPM : n;
    for (int64_t i = (int64_t)block * 8 + (threadIdx.x >> 5); i < end; i += (int64_t)t.blocks * 8) {
        const bool there = i < n;
        const int64_t r = there ? source_row(s, i) : 0;
        const T *x = static_cast<const T *>(s.src) + r * s.ld;
        if (is_x && there && lane == 0) pick.label[i] = (int)pick.labels[r];
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
            if (lane == 0) t.row_down[i] = down;
        }
        for (int k = lane; k < t.row.ld; k += 32) {
            const bool in = there && k < s.K;
            const int64_t at = i * t.row.ld + k;
            if (SPLIT) {
                const float v = in ? to_f32<T>(x[k]) : 0.f;
                store_split(t.row, at, v, up, 1.0f);
                if (t.col.p) {
                    float cup = 1.f, cdown;
                    if (k < s.K) plane_scale(__uint_as_float(__ldg(t.largest + k)), cup, cdown);
                    store_split(t.col, at, v, cup, kSecondPlane);
                }
            } else {
                t.row.p[at] = in ? reinterpret_cast<const uint16_t *>(x)[k] : (uint16_t)0;
            }
        }
    }
}

__device__ __forceinline__ void join_stats(float &mx, float &sum, float2 v)
{
    const float top = fmaxf(mx, v.x), ref = top == -INFINITY ? 0.f : top;
    sum = sum * exp2_fast(mx - ref) + v.y * exp2_fast(v.x - ref);
    mx = top;
}

// lse of the rows of a chunk from the parts of their tiles: eight rows a block, the parts dealt over 128 groups of eight
// threads.  The sum of their losses goes to loss_part; the block that comes last of all chunks adds those up, in their order.
constexpr int kJoinRows = 8;

struct NllJoin {
    const float2 *stats;
    int parts, row0, row_cap;
    const int *rows, *total;
    const float *picked2;
    float *lse2, *lse_out, *loss_part;  // loss_part: of this chunk
    const float *all_parts;
    int all_count;
    float inv_count;
    int *joined;
    const int *failed;
    float *loss;
};

__global__ void __launch_bounds__(1024) nll_join_kernel(const NllJoin a)
{
    __shared__ float2 red[32][kJoinRows];
    __shared__ float total[32];
    __shared__ bool last;
    let_next_kernel_start();
    wait_for_kernels_before();
    const int lane = threadIdx.x & 31, g = threadIdx.x >> 5, row = threadIdx.x % kJoinRows;
    const int i = blockIdx.x * kJoinRows + row;  // of the chunk
    const bool on = i < a.row_cap && a.row0 + i < *a.total;
    float mx = -INFINITY, sum = 0.f;
    if (on) {
#pragma unroll 4
        for (int p = threadIdx.x / kJoinRows; p < a.parts; p += 1024 / kJoinRows) join_stats(mx, sum, a.stats[(int64_t)p * a.row_cap + i]);
    }
    // the four groups of a warp, then the 32 warps, in trees: the same for every number of parts
#pragma unroll
    for (int o = 16; o >= kJoinRows; o >>= 1) join_stats(mx, sum, make_float2(__shfl_xor_sync(FULL, mx, o), __shfl_xor_sync(FULL, sum, o)));
    if (lane < kJoinRows) red[g][row] = make_float2(mx, sum);
    __syncthreads();
    if (g < kJoinRows) {  // warp g: row g of the block
        const float2 mine = red[lane][g];
        mx = mine.x, sum = mine.y;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) join_stats(mx, sum, make_float2(__shfl_xor_sync(FULL, mx, o), __shfl_xor_sync(FULL, sum, o)));
        const int r = blockIdx.x * kJoinRows + g;
        if (lane == 0) {
            float loss = 0.f;
            if (r < a.row_cap && a.row0 + r < *a.total) {
                const float l = mx + log2f(sum);
                a.lse2[r] = l;
                if (a.lse_out) a.lse_out[a.rows[a.row0 + r]] = l * kLn2;
                loss = (l - a.picked2[r]) * kLn2;
            }
            total[g] = loss;
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        float loss = 0.f;
        for (int r = 0; r < kJoinRows; ++r) loss += total[r];
        a.loss_part[blockIdx.x] = loss;
        __threadfence();
        last = atomicAdd(a.joined, 1) == a.all_count - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    float s = 0.f;
    for (int p = threadIdx.x; p < a.all_count; p += 1024) s += __ldcg(a.all_parts + p);
    s = all_sum(s);
    if (lane == 0) total[g] = s;
    __syncthreads();
    if (g == 0) {
        s = all_sum(total[lane]);
        if (lane == 0) *a.loss = *a.failed ? __int_as_float(0x7fffffff) : s * a.inv_count;
    }
}

// ---- what is left once the products are done: three independent sums, in one launch ----
// WARPS warps a block: 8, or 32 for the bias sums of many rows, at 32 registers so that two blocks fit an SM (16k x 64k x 512 bf16:
// 4.38 ms in all; 4.65 with 8 warps, 4.44 with one block an SM).
// gx of the listed rows of a chunk: the partial sums of the splits, scaled back; NaN when a wait gave up before.  With many splits
// (`dealt`) a block has one row and 32 columns, and its warps share the splits; otherwise a warp has a row.
struct RowsOut {
    const float *acc;
    int64_t ld, split;
    int splits, row0, row_cap, K;
    const int *rows, *total, *failed;
    float scale;
    const unsigned *largest;
    void *gx;
    int64_t ldgx;
    float *loss;
    bool dealt;
    int blocks_x, blocks_y;
};
// gb of a piece from the sums over 32 rows of a chunk, onto those of the chunks before (acc); the last chunk writes the result.
// 32 classes a block, the sums dealt over its warps; with few rows (not `dealt`) a thread adds up a class alone.
struct BiasOut {
    const float *part;
    int64_t ld;
    int row0, row_cap, count;
    const int *total;
    float scale;
    float *acc;
    bool first, last, f32;
    void *gb;
    bool dealt;
    int blocks;
};
// gw from the partial sums of the splits (and of all chunks)
struct WeightsOut {
    const float *acc;
    int64_t ld, split, C, ldgw;
    int splits, K;
    float scale;
    const unsigned *largest;
    void *gw;
    int blocks;
};

// One row of a result by a warp, from the partial sums of the splits; four columns a lane at a time, loads of several splits
// on their way together.
template <class T>
__device__ __forceinline__ void sum_splits(const float *acc, int64_t split, int splits, int K, float scale, const unsigned *largest, bool bad, T *out)
{
    for (int k0 = threadIdx.x & 31; k0 < K; k0 += 128) {
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int s = 0; s < splits; ++s) {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += k0 + 32 * j < K ? acc[s * split + k0 + 32 * j] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = k0 + 32 * j;
            if (k >= K) break;
            float up, down = 1.f;
            if (largest != nullptr) plane_scale(__uint_as_float(__ldg(largest + k)), up, down);
            out[k] = from_f32<T>(bad ? __int_as_float(0x7fffffff) : v[j] * scale * down);
        }
    }
}

template <class T, int WARPS>
__device__ __forceinline__ void rows_out(const RowsOut &a, int block, float (&red)[WARPS][33])
{
    const int lane = threadIdx.x & 31, g = threadIdx.x >> 5, bx = block % a.blocks_x;
    const bool bad = *a.failed != 0;
    if (bad && block == 0 && threadIdx.x == 0) *a.loss = __int_as_float(0x7fffffff);
    const int left = *a.total - a.row0, count = left < a.row_cap ? left : a.row_cap;
    if (!a.dealt) {
        for (int i = bx * WARPS + g; i < count; i += a.blocks_x * WARPS)
            sum_splits<T>(a.acc + (int64_t)i * a.ld, a.split, a.splits, a.K, a.scale, a.largest, bad,
                          static_cast<T *>(a.gx) + (int64_t)a.rows[a.row0 + i] * a.ldgx);
        return;
    }
    const int k = block / a.blocks_x * 32 + lane;
    for (int i = bx; i < count; i += a.blocks_x) {
        float v = 0.f;
        if (k < a.K) {
#pragma unroll 4
            for (int s = g; s < a.splits; s += WARPS) v += a.acc[s * a.split + (int64_t)i * a.ld + k];
        }
        __syncthreads();
        red[g][lane] = v;
        __syncthreads();
        if (g != 0 || k >= a.K) continue;
        for (int w = 1; w < WARPS; ++w) v += red[w][lane];
        float up, down = 1.f;
        if (a.largest != nullptr) plane_scale(__uint_as_float(__ldg(a.largest + k)), up, down);
        static_cast<T *>(a.gx)[(int64_t)a.rows[a.row0 + i] * a.ldgx + k] = from_f32<T>(bad ? __int_as_float(0x7fffffff) : v * a.scale * down);
    }
}

template <class T, int WARPS>
__device__ __forceinline__ void bias_out(const BiasOut &a, int block, float (&red)[WARPS][33])
{
    const int lane = threadIdx.x & 31, g = threadIdx.x >> 5, c = a.dealt ? block * 32 + lane : block * WARPS * 32 + threadIdx.x;
    int rows = *a.total - a.row0;
    rows = rows < 0 ? 0 : rows < a.row_cap ? rows : a.row_cap;
    const int groups = (rows + kPM - 1) / kPM * (kPM / 32);  // whole tiles have been written
    float s = 0.f;
    if (c < a.count) {
#pragma unroll 8
        for (int i = a.dealt ? g : 0; i < groups; i += a.dealt ? WARPS : 1) s += a.part[(int64_t)i * a.ld + c];
    }
    if (a.dealt) {
        red[g][lane] = s;
        __syncthreads();
        if (g != 0) return;
        for (int w = 1; w < WARPS; ++w) s += red[w][lane];
    }
    if (c >= a.count) return;
    if (!a.first) s += a.acc[c];
    if (!a.last) a.acc[c] = s;
    else if (a.f32) static_cast<float *>(a.gb)[c] = s * a.scale;
    else static_cast<T *>(a.gb)[c] = from_f32<T>(s * a.scale);
}

template <class T, int WARPS>
__device__ __forceinline__ void weights_out(const WeightsOut &a, int block)
{
    for (int64_t c = (int64_t)block * WARPS + (threadIdx.x >> 5); c < a.C; c += (int64_t)a.blocks * WARPS)
        sum_splits<T>(a.acc + c * a.ld, a.split, a.splits, a.K, a.scale, a.largest, false, static_cast<T *>(a.gw) + c * a.ldgw);
}

// The first blocks sum up rows, the next ones the bias, the rest weights; none of a kind whose `blocks` are 0.
template <class T, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 64 / WARPS) nll_out_kernel(const RowsOut r, const BiasOut b, const WeightsOut w)
{
    __shared__ float red[WARPS][33];
    let_next_kernel_start();
    wait_for_kernels_before();
    const int rows_blocks = r.blocks_x * r.blocks_y, block = (int)blockIdx.x;
    if (block < rows_blocks) rows_out<T, WARPS>(r, block, red);
    else if (block < rows_blocks + b.blocks) bias_out<T, WARPS>(b, block - rows_blocks, red);
    else weights_out<T, WARPS>(w, block - rows_blocks - b.blocks);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// G of a chunk and a piece, elements of 16 bits (336 MB).  Measured for 16k rows, 64k classes, 512 features in bf16, the
// products alone: 5.0 ms with 20 M elements, 4.5 with 45 M, 4.29 with 90 M, 4.26 with 180 M, 4.13 with 360 M: fewer and longer
// launches win over a G that stays in the L2 cache.
constexpr int64_t kNllPieceElements = 160ll << 20;

static int64_t round_up(int64_t v, int64_t to) { return ceil_div(v, to) * to; }

// Time of the products of one kind on all SMs, in ns: `tiles` results of `blocks` reduction steps each, split s ways, and
// the partial sums (`result` bytes a split) that then have to be written.  A step is 0.4 us at the rate the products reach.
static double nll_product_ns(int64_t tiles, int64_t blocks, int64_t s, int products, double result)
{
    return (double)ceil_div(tiles * s, sm_count()) * (double)ceil_div(blocks, s) * 400.0 * products + (double)s * result / 4000.0;
}

static int nll_splits(int64_t tiles, int64_t blocks, int products, double result, double *ns)
{
    int64_t most = blocks / 4 < 148 ? blocks / 4 : 148, best = 1;
    *ns = nll_product_ns(tiles, blocks, 1, products, result);
    for (int64_t s = 2; s <= most && tiles * s <= 8 * sm_count(); ++s) {
        const double t = nll_product_ns(tiles, blocks, s, products, result);
        if (t < *ns) *ns = t, best = s;
    }
    return (int)best;
}

struct NllPlan {
    int planes;
    int64_t blocks, padded, row_cap, chunks, cls_padded, piece, ld, acc_ld;
    int row_splits, weight_splits;
    bool copy_w, direct, together;
    size_t counts, rows, total, failed, joined, label, picked2, lse2, loss_part, bias2, stats;
    size_t x_row, x_col, w_row, w_col, x_down, w_down, largest;
    size_t grad, acc_x, acc_w, bias_part, bias_acc, bytes;
};

// Rows in chunks, classes in pieces, reductions in splits: of the chunk sizes up to 128 tiles the one whose modelled time is
// least.  Few long chunks add up gw less often, short ones leave longer pieces and add up gx less often, and the tiles of
// the two products should fill whole rounds of the SMs.
static void nll_divide(NllPlan &p, int64_t K, int64_t C, bool may_direct)
{
    const int64_t tiles = p.padded / kPM, tiles_k = ceil_div(K, kPN), cls_tiles = p.cls_padded / kPN;
    const int products = p.planes == 2 ? 3 : 1;
    const int64_t area = kNllPieceElements / p.planes / (kPM * kPN);  // tiles of G
    double best = 0;
    for (int64_t t = tiles < 128 ? tiles : 128; t >= 1; --t) {
        const int64_t chunks = ceil_div(tiles, t);
        if (t != ceil_div(tiles, chunks)) continue;  // not the even division into that many chunks
        int64_t piece = area / t < 1 ? 1 : area / t < cls_tiles ? area / t : cls_tiles;
        const int64_t pieces = ceil_div(cls_tiles, piece);
        piece = ceil_div(cls_tiles, pieces);
        double rows_ns, weights_ns;
        const double x_bytes = (double)t * kPM * K * 4, w_bytes = (double)piece * kPN * K * 4;
        const int rs = nll_splits(t * tiles_k, piece * (kPN / kPK), products, pieces > 1 ? 2 * x_bytes : x_bytes, &rows_ns);
        const int ws = nll_splits(2 * piece * tiles_k, t * (kPM / kPK), products, chunks > 1 ? 2 * w_bytes : w_bytes, &weights_ns);
        const bool direct = may_direct && chunks == 1 && ws == 1;
        const double logits_ns = (double)ceil_div(t * piece, sm_count()) * (double)ceil_div(K, kPK) * 400.0 * products;
        const double ns = (double)(chunks * pieces) * (rows_ns + weights_ns + logits_ns + 9000.0) +
                          (direct ? 0.0 : (double)ws * C * K * 4 / 4000.0) + (double)chunks * rs * x_bytes / 4000.0;
        if (best == 0 || ns < best) {
            best = ns;
            p.row_cap = t * kPM, p.chunks = chunks, p.piece = piece * kPN, p.row_splits = rs, p.weight_splits = ws, p.direct = direct;
            // One launch: 300 x 30000 x 256 bf16 in 97 us instead of 109, 5003 x 20011 x 200 fp32 in 598 instead of 624 (with
            // the sums in one launch too); 16k x 64k x 512 bf16, where the rule keeps them apart, in 4.65 ms instead of 4.37.
            p.together = rows_ns + weights_ns < 150e3;
        }
        if (tiles <= 8) break;  // a small call: one chunk, and no search
    }
}

// `copy_w`: bf16 weights whose rows TMA cannot read where they are.  `may_direct`: gw's rows can be written by TMA.
static NllPlan nll_plan(int dtype, int64_t n, int64_t K, int64_t C, bool grad, bool copy_w, bool may_direct)
{
    NllPlan p{};
    const bool f32 = dtype == SGNN_F32;
    p.planes = f32 ? 2 : 1;
    p.copy_w = f32 || copy_w;
    p.blocks = ceil_div(n, kListRows);
    p.padded = round_up(n, kPM);
    p.cls_padded = round_up(C, kPN);
    p.ld = round_up(K, 8);
    p.acc_ld = round_up(K, 32);
    nll_divide(p, K, C, may_direct);
    size_t at = 0;
    const auto take = [&at](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    const size_t mat_x = (size_t)p.planes * p.padded * p.ld * 2, mat_w = (size_t)p.planes * C * p.ld * 2;
    p.counts = take(p.blocks * 4), p.rows = take(n * 4), p.total = take(4), p.failed = take(4), p.joined = take(4);
    p.label = take(p.padded * 4), p.picked2 = take(p.padded * 4), p.lse2 = take(p.row_cap * 4);
    p.loss_part = take(p.chunks * p.row_cap / kJoinRows * 4), p.bias2 = take(p.cls_padded * 4);
    p.stats = take((size_t)p.cls_padded / 128 * p.row_cap * 8);
    p.x_row = take(mat_x), p.w_row = take(p.copy_w ? mat_w : 0);
    if (f32) {
        p.x_down = take(p.padded * 4), p.w_down = take(p.cls_padded * 4);
        if (grad) p.x_col = take(mat_x), p.w_col = take(mat_w), p.largest = take(2 * K * 4);
    }
    if (grad) {
        p.grad = take((size_t)p.planes * p.row_cap * p.piece * 2);
        p.acc_x = take((size_t)p.row_splits * p.row_cap * p.acc_ld * 4);
        p.acc_w = take(p.direct ? 0 : (size_t)p.weight_splits * C * p.acc_ld * 4);
        p.bias_part = take((size_t)p.row_cap / 32 * p.piece * 4);
        p.bias_acc = take(p.chunks > 1 ? (size_t)C * 4 : 0);
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
static bool nll_may_direct(int dtype, const void *gw, int64_t ldgw)
{
    return aligned16(gw) && ldgw * (int64_t)elem_bytes(dtype) % 16 == 0;
}

template <int KIND, int PLANES, int CTAS>
static int nll_product_blocks(const ProductCall &c, const ProductCall &c2, int64_t units, cudaStream_t s)
{
    constexpr int smem = product_shared_bytes<KIND, PLANES, CTAS>();
    static ResidentCache cache;
    int resident = 0, rc = resident_blocks(nll_product_kernel<KIND, PLANES, CTAS>, kPThreads, smem, smem, cache, &resident);
    if (rc) return rc;
    const int64_t most = resident / CTAS, grid = CTAS * (units < most ? units : most);
    SGNN_CUDA_OK(launch_clusters(CTAS, nll_product_kernel<KIND, PLANES, CTAS>, dim3((unsigned)grid), kPThreads, smem, s, c, c2));
    return SGNN_OK;
}

// Two blocks a result?  They need a third less of their operands from L2, which bounds the gradients and the fp32 logits (16k x
// 64k x 512 bf16: gx 1313 -> 989 us, gw 1490 -> 1259 us; the fp32 loss alone, 5003 rows and 20011 classes: over 200 features 174 ->
// 139 us, over 1000 840 -> 668, between them, at 512, 314 -> 333); the bf16 logits wait for their exponentials (779 against 789 us),
// and few rows are better spread over more blocks (300 x 30000 x 256 bf16, all of it: 104 against 130 us).
template <int KIND, int PLANES>
constexpr bool kNllPairs = PLANES == 2 || !nll_is_logits(KIND);
static bool nll_in_pairs(int64_t row_cap) { return row_cap > 1024; }

// Results of `rows` rows at most and `tiles` beside each other (gradients: and of `rows2` and `tiles2`; splits count as tiles)
template <int KIND, int PLANES>
static int nll_product(const ProductCall &c, const ProductCall &c2, int64_t rows, int64_t tiles, int64_t rows2, int64_t tiles2, cudaStream_t s)
{
    if constexpr (kNllPairs<KIND, PLANES>) {
        if (nll_in_pairs(c.row_cap))
            return nll_product_blocks<KIND, PLANES, 2>(c, c2, ceil_div(rows, 2 * kPM) * tiles + ceil_div(rows2, 2 * kPM) * tiles2, s);
    }
    return nll_product_blocks<KIND, PLANES, 1>(c, c2, ceil_div(rows, kPM) * tiles + ceil_div(rows2, kPM) * tiles2, s);
}

// fp32 logits over more features than this: sums of their own for the cross products of the planes, and the main sums move on into
// registers every 512.  Every addition in tensor memory rounds towards zero, and with all three products in one sum a logit over
// 512 features has 96 of them, 32 so: gradients over 16 to 300 classes come out 0.4e-6 to 0.8e-6 off instead of 1.0e-6 to 1.4e-6
// (and over 256 features 0.7e-6 either way).  One result in tensor memory at a time is the price: 5003 x 512 x 20011 with gradients
// 1.42 ms against 1.26, the loss alone 327 us against 268; 100 x 2048 x 30000, with several windows, 0.76 ms against 0.79.
constexpr int64_t kNllShortFeatures = 256;
static bool nll_logits_long(int64_t K) { return K > kNllShortFeatures; }

template <int SHORT, int LONG, int PLANES>
static int nll_logits(const ProductCall &c, int64_t rows, int64_t tiles, cudaStream_t s)
{
    if constexpr (PLANES == 2) {
        if (nll_logits_long(c.feats)) return nll_product<LONG, PLANES>(c, c, rows, tiles, 0, 0, s);
    }
    return nll_product<SHORT, PLANES>(c, c, rows, tiles, 0, 0, s);
}

template <class T, int PLANES>
static int nll_run(const NllCall &c, const NllPlan &p)
{
    constexpr bool f32 = PLANES == 2;
    const bool grad = c.gx != nullptr;
    const auto ints = [&](size_t at) { return reinterpret_cast<int *>(c.ws + at); };
    const auto floats = [&](size_t at) { return reinterpret_cast<float *>(c.ws + at); };
    const auto halves = [&](size_t at) { return reinterpret_cast<uint16_t *>(c.ws + at); };
    const int64_t wide = 16 * sm_count();
    const auto blocks = [wide](int64_t warps) { return (unsigned)(ceil_div(warps, 8) < wide ? ceil_div(warps, 8) : wide); };
    cudaStream_t s = c.s;
    int rc;

    // the rows in the loss, and what later kernels start from
    if (p.blocks > 1) {
        SGNN_CUDA_OK(launch_chained(nll_count_kernel, dim3((unsigned)p.blocks), kListThreads, 0, s, c.labels, c.mask, c.n, c.C, ints(p.counts)));
    }
    const bool cols = f32 && grad;
    unsigned *largest = cols ? reinterpret_cast<unsigned *>(c.ws + p.largest) : nullptr;
    const NllStart start{c.labels, c.mask, c.n, c.C, p.cls_padded, ints(p.counts), ints(p.rows), ints(p.total), (int)p.blocks, c.bias,
                         floats(p.bias2), f32 ? floats(p.w_down) : nullptr, c.lse, ints(p.failed), ints(p.joined), largest, (int)c.K,
                         grad ? c.gx : nullptr, c.ldgx};
    const int64_t cleared = p.cls_padded + (c.lse ? c.n : 0) + (grad ? c.n * c.K / 8 : 0);
    SGNN_CUDA_OK(launch_chained(nll_start_kernel<T>, dim3((unsigned)p.blocks + blocks(ceil_div(cleared, 32))), kListThreads, 0, s, start));

    // the operands as the products read them
    TakeSide xs{RowSource{c.x, c.ldx, ints(p.rows), ints(p.total), 0, (int)c.K},
                Planes{halves(p.x_row), p.ld, p.padded * p.ld},
                Planes{cols ? halves(p.x_col) : nullptr, p.ld, p.padded * p.ld},
                largest, f32 ? floats(p.x_down) : nullptr, (int)blocks(p.padded)};
    TakeSide ws{RowSource{c.w, c.ldw, nullptr, nullptr, c.C, (int)c.K},
                Planes{halves(p.w_row), p.ld, c.C * p.ld},
                Planes{cols ? halves(p.w_col) : nullptr, p.ld, c.C * p.ld},
                cols ? largest + c.K : nullptr, f32 ? floats(p.w_down) : nullptr, p.copy_w ? (int)blocks(c.C) : 0};
    if (cols) {
        const int64_t rows = c.n > c.C ? c.n : c.C, tall = ceil_div(rows, 64) < 2 * sm_count() ? ceil_div(rows, 64) : 2 * sm_count();
        SGNN_CUDA_OK(launch_chained(nll_column_max_kernel, dim3((unsigned)ceil_div(c.K, 32), (unsigned)tall, 2), 256, 0, s, xs.src, ws.src, largest));
    }
    SGNN_CUDA_OK(launch_chained(nll_take_kernel<T, f32>, dim3((unsigned)(xs.blocks + ws.blocks)), 256, 0, s, xs, ws,
                                Picked{c.labels, ints(p.label)}));

    // tensor maps: x and W along k (rows of a tile at once) and across it (64 steps of the reduction at once), G likewise
    ProductCall lc{}, xc{}, wc{};
    const void *wp = p.copy_w ? (const void *)ws.row.p : c.w;
    const int64_t wld = p.copy_w ? p.ld : c.ldw, wst = p.copy_w ? ws.row.stride : c.C * c.ldw;
    if ((rc = umma_tensor_map(&lc.a, xs.row.p, !f32, c.K, p.padded, p.ld, PLANES, xs.row.stride, kPM))) return rc;
    const bool pairs = kNllPairs<kLogitStats, PLANES> && nll_in_pairs(p.row_cap);  // each of the two reads half of a tile's classes
    if ((rc = umma_tensor_map(&lc.b, wp, !f32, c.K, c.C, wld, PLANES, wst, pairs ? kPN / 2 : kPN))) return rc;
    lc.total = ints(p.total), lc.failed = ints(p.failed), lc.feats = (int)c.K, lc.splits = 1, lc.bf16 = !f32;
    lc.bias2 = floats(p.bias2), lc.row_scale = xs.row_down, lc.cls_scale = ws.row_down, lc.classes = c.C;
    lc.stats = reinterpret_cast<float2 *>(c.ws + p.stats), lc.row_cap = (int)p.row_cap, lc.lse2 = floats(p.lse2);
    lc.scale = c.inv_count * (f32 ? 1.0f / kGradScale : 1.0f);
    const int64_t x_split = p.row_cap * p.acc_ld, w_split = c.C * p.acc_ld;
    if (grad) {
        lc.bias_part = c.gb ? floats(p.bias_part) : nullptr, lc.grad_ld = p.piece;
        xc = lc, wc = lc;
        uint16_t *g = halves(p.grad);
        const int64_t plane = p.row_cap * p.piece;
        if ((rc = umma_store_map(&lc.o, g, f32 ? StoreType::kF16 : StoreType::kBf16, p.piece, p.row_cap, p.piece, PLANES, plane, f32 ? 32 : 64))) return rc;
        if ((rc = umma_tensor_map(&xc.a, g, !f32, p.piece, p.row_cap, p.piece, PLANES, plane, kPM))) return rc;
        if ((rc = umma_tensor_map(&xc.b, f32 ? (const void *)ws.col.p : wp, !f32, c.K, c.C, wld, PLANES, wst, kPK))) return rc;
        if ((rc = umma_store_map(&xc.o, floats(p.acc_x), StoreType::kF32, p.acc_ld, p.row_cap, p.acc_ld, p.row_splits, x_split, 32))) return rc;
        if ((rc = umma_tensor_map(&wc.a, g, !f32, p.piece, p.row_cap, p.piece, PLANES, plane, kPK))) return rc;
        if ((rc = umma_tensor_map(&wc.b, f32 ? xs.col.p : xs.row.p, !f32, c.K, p.padded, p.ld, PLANES, xs.row.stride, kPK))) return rc;
        xc.splits = p.row_splits, wc.splits = p.weight_splits;
        wc.direct = p.direct, wc.direct_bf16 = !f32, wc.col_largest = largest;
        if (p.direct) {
            rc = umma_store_map(&wc.o, c.gw, f32 ? StoreType::kF32 : StoreType::kBf16, c.K, c.C, c.ldgw, 1, c.C * c.ldgw, f32 ? 32 : 64);
        } else {
            rc = umma_store_map(&wc.o, floats(p.acc_w), StoreType::kF32, p.acc_ld, c.C, p.acc_ld, p.weight_splits, w_split, 32);
        }
        if (rc) return rc;
    }
    const int64_t tiles_k = ceil_div(c.K, kPN), join_blocks = p.row_cap / kJoinRows;
    for (int64_t q = 0; q < p.chunks; ++q) {
        const int row0 = (int)(q * p.row_cap);
        for (ProductCall *k : {&lc, &xc, &wc}) k->row0 = row0;
        lc.label = ints(p.label) + row0, lc.picked2 = floats(p.picked2) + row0;
        lc.cls0 = 0, lc.cls_count = (int)c.C;
        if ((rc = nll_logits<kLogitStats, kLongStats, PLANES>(lc, p.row_cap, ceil_div(c.C, kPN), s))) return rc;
        const NllJoin join{lc.stats, (int)(p.cls_padded / 128), row0, (int)p.row_cap, ints(p.rows), ints(p.total), lc.picked2,
                           floats(p.lse2), c.lse, floats(p.loss_part) + q * join_blocks, floats(p.loss_part),
                           (int)(p.chunks * join_blocks), c.inv_count, ints(p.joined), ints(p.failed), c.loss};
        SGNN_CUDA_OK(launch_chained(nll_join_kernel, dim3((unsigned)join_blocks), 1024, 0, s, join));
        if (!grad) continue;
        for (int64_t first = 0; first < c.C; first += p.piece) {
            const int64_t count = c.C - first < p.piece ? c.C - first : p.piece;
            for (ProductCall *k : {&lc, &xc, &wc}) k->cls0 = (int)first, k->cls_count = (int)count;
            if ((rc = nll_logits<kLogitGrad, kLongGrad, PLANES>(lc, p.row_cap, ceil_div(count, kPN), s))) return rc;
            xc.add = first > 0, wc.add = q > 0;
            if (p.together) {
                if ((rc = nll_product<kGradients, PLANES>(xc, wc, p.row_cap, tiles_k * p.row_splits, count, tiles_k * p.weight_splits, s))) return rc;
            } else {
                if ((rc = nll_product<kRowGrad, PLANES>(xc, xc, p.row_cap, tiles_k * p.row_splits, 0, 0, s))) return rc;
                if ((rc = nll_product<kWeightGrad, PLANES>(wc, wc, count, tiles_k * p.weight_splits, 0, 0, s))) return rc;
            }
            const bool deal = p.row_cap > 256;
            const int warps = p.row_cap >= 8192 ? 32 : 8;
            BiasOut bias{};
            if (c.gb) {
                char *gb = static_cast<char *>(c.gb) + first * (c.bias.f32 ? 4 : sizeof(T));
                bias = BiasOut{lc.bias_part, p.piece, row0, (int)p.row_cap, (int)count, ints(p.total), lc.scale,
                               p.chunks > 1 ? floats(p.bias_acc) + first : nullptr, q == 0, q + 1 == p.chunks, c.bias.f32, gb, deal,
                               (int)ceil_div(count, deal ? 32 : 32 * warps)};
            }
            const bool last = first + p.piece >= c.C;  // the pieces of this chunk are all in gx
            RowsOut rows{};
            if (last) {
                const bool dealt = p.row_splits >= 8;
                rows = RowsOut{floats(p.acc_x), p.acc_ld, x_split, p.row_splits, row0, (int)p.row_cap, (int)c.K, ints(p.rows), ints(p.total),
                               ints(p.failed), lc.scale, cols ? largest + c.K : nullptr, c.gx, c.ldgx, c.loss, dealt,
                               dealt ? (int)(p.row_cap < wide ? p.row_cap : wide) : (int)ceil_div(p.row_cap, warps),
                               dealt ? (int)ceil_div(c.K, 32) : 1};
            }
            WeightsOut weights{};
            if (last && q + 1 == p.chunks && !p.direct)
                weights = WeightsOut{floats(p.acc_w), p.acc_ld, w_split, c.C, c.ldgw, p.weight_splits, (int)c.K, lc.scale, largest, c.gw,
                                     (int)(ceil_div(c.C, warps) < wide ? ceil_div(c.C, warps) : wide)};
            const int grid = rows.blocks_x * rows.blocks_y + bias.blocks + weights.blocks;
            if (grid > 0)
                SGNN_CUDA_OK(launch_chained(warps == 32 ? nll_out_kernel<T, 32> : nll_out_kernel<T, 8>, dim3((unsigned)grid), warps * 32, 0, s,
                                            rows, bias, weights));
        }
    }
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
    *bytes = 0;
    if (n > 0) {  // enough for every layout of the weights: a copy of them, gw written directly or not
        const size_t added = nll_plan(dtype, n, K, C, with_grad != 0, true, false).bytes;
        const size_t direct = nll_plan(dtype, n, K, C, with_grad != 0, true, true).bytes;
        *bytes = added > direct ? added : direct;
    }
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
    const auto on = [](const void *p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; };
    SGNN_REQUIRE(on(d_x, b) && on(d_w, b) && on(d_gx, b) && on(d_gw, b) && on(d_bias, elem_bytes(bias_dtype)) &&
                     on(d_gb, elem_bytes(bias_dtype)) && on(d_labels, 8) && on(d_loss, 4) && on(d_lse, 4),
                 SGNN_ERR_INVALID_ARGUMENT, "%s: pointers must be aligned to their element", who);
    const NllPlan p = nll_plan(dtype, n, K, C, d_gx != nullptr, nll_must_copy_weights(dtype, d_w, ldw, C),
                               nll_may_direct(dtype, d_gw, ldgw));
    SGNN_REQUIRE(d_workspace != nullptr && workspace_bytes >= p.bytes && reinterpret_cast<uintptr_t>(d_workspace) % 256 == 0,
                 SGNN_ERR_WORKSPACE, "%s: 256-byte aligned workspace of %zu bytes needed, %zu given", who, p.bytes, workspace_bytes);
    const NllCall c{dtype, d_x, ldx, d_w, ldw, NllBias{d_bias, bias_dtype == SGNN_F32}, d_labels, d_mask, inv_count, n, K, C, d_loss,
                    d_lse, d_gx, ldgx, d_gw, ldgw, d_gb, static_cast<char *>(d_workspace), s};
    return dtype == SGNN_F32 ? nll_run<float, 2>(c, p) : nll_run<__nv_bfloat16, 1>(c, p);
}
