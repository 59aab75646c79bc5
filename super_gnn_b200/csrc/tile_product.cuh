// C[m, n] = sum_k A(m, k) B(n, k) in fp32, operands and result through functors: one 64 x 64 tile a block, 4 x 4
// values a thread, 16 steps of k staged in shared memory.  blockIdx.z splits k into equal ranges.
#pragma once
#include "common.cuh"

namespace sgnn {

constexpr int kTile = 64, kTileK = 16, kTileThreads = 256;

template <class LA, class LB, class EP>
__global__ void __launch_bounds__(kTileThreads)
tile_product_kernel(LA a, LB b, EP ep, int64_t K, int64_t k_per_split)
{
    __shared__ float sa[kTileK][kTile + 1], sb[kTileK][kTile + 1];
    const int64_t m0 = (int64_t)blockIdx.y * kTile, n0 = (int64_t)blockIdx.x * kTile;
    const int64_t k_begin = (int64_t)blockIdx.z * k_per_split;
    int64_t k_end = k_begin + k_per_split;
    if (k_end > K) k_end = K;
    const int tm = threadIdx.x / 16, tn = threadIdx.x % 16;
    float acc[4][4] = {};
    for (int64_t k0 = k_begin; k0 < k_end; k0 += kTileK) {
        for (int i = threadIdx.x; i < kTile * kTileK; i += kTileThreads) {
            const int mm = i / kTileK, kk = i % kTileK;
            const bool in = k0 + kk < k_end;
            sa[kk][mm] = in ? a(m0 + mm, k0 + kk) : 0.f;
            sb[kk][mm] = in ? b(n0 + mm, k0 + kk) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < kTileK; ++kk) {
            float x[4], y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = sa[kk][tm * 4 + i], y[i] = sb[kk][tn * 4 + i];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] += x[i] * y[j];
        }
        __syncthreads();
    }
    ep(m0 + tm * 4, n0 + tn * 4, acc, (int)blockIdx.z);
}

}  // namespace sgnn
