// answers_planes.hip -- a network's answers between the rows its kernels work on and the planes of MedicalVolumes.
#include "answers.h"

namespace qmri {
// K values a pixel, rows (S, P, K) <-> planes (K, P, S) as MedicalVolumes hold them.  Labels are int32 with -1 for "none" in rows,
// uint8 with 255 in planes.
__device__ __forceinline__ float plane_value(float v) { return v; }
__device__ __forceinline__ unsigned char plane_value(int v) { return v < 0 ? 255 : (unsigned char)v; }
__device__ __forceinline__ void row_value(float v, float &o) { o = v; }
__device__ __forceinline__ void row_value(unsigned char v, int &o) { o = v == 255 ? -1 : v; }
__device__ __forceinline__ void row_value(unsigned char v, unsigned char &o) { o = v; }
template <typename R, typename V>
__global__ __launch_bounds__(256) void rows_to_planes_kernel(const R *__restrict__ x, long long P, int S, int K, V *__restrict__ y) {
    __shared__ V tile[32][33];
    const long long p0 = (long long)blockIdx.x * 32;
    const int s0 = blockIdx.y * 32, k = blockIdx.z;
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;  // 32 x 8
    for (int r = ty; r < 32; r += 8) {
        const int s = s0 + r;
        const long long p = p0 + tx;
        if (s < S && p < P) tile[r][tx] = plane_value(x[((long long)s * P + p) * K + k]);
    }
    __syncthreads();
    for (int r = ty; r < 32; r += 8) {
        const long long p = p0 + r;
        const int s = s0 + tx;
        if (p < P && s < S) y[((long long)k * P + p) * S + s] = tile[tx][r];
    }
}
template <typename V, typename R>
__global__ __launch_bounds__(256) void planes_to_rows_kernel(const V *__restrict__ x, long long P, int S, int K, R *__restrict__ y) {
    __shared__ R tile[32][33];
    const long long p0 = (long long)blockIdx.x * 32;
    const int s0 = blockIdx.y * 32, k = blockIdx.z;
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    for (int r = ty; r < 32; r += 8) {
        const long long p = p0 + r;
        const int s = s0 + tx;
        if (p < P && s < S) row_value(x[((long long)k * P + p) * S + s], tile[r][tx]);
    }
    __syncthreads();
    for (int r = ty; r < 32; r += 8) {
        const int s = s0 + r;
        const long long p = p0 + tx;
        if (s < S && p < P) y[((long long)s * P + p) * K + k] = tile[tx][r];
    }
}
hipError_t rows_to_planes_launch(const void *x, int is_label, long long P, int S, int K, void *y, hipStream_t stream) {
    (void)hipGetLastError();
    const dim3 grid((unsigned)((P + 31) / 32), (unsigned)((S + 31) / 32), (unsigned)K), block(256);
    if (is_label)
        hipLaunchKernelGGL((rows_to_planes_kernel<int, unsigned char>), grid, block, 0, stream, static_cast<const int *>(x), P, S, K,
                           static_cast<unsigned char *>(y));
    else
        hipLaunchKernelGGL((rows_to_planes_kernel<float, float>), grid, block, 0, stream, static_cast<const float *>(x), P, S, K,
                           static_cast<float *>(y));
    return hipGetLastError();
}
// kind 0: float32; 1: labels, uint8 rows; 2: labels, int32 rows
hipError_t planes_to_rows_launch(const void *x, int kind, long long P, int S, int K, void *y, hipStream_t stream) {
    (void)hipGetLastError();
    const dim3 grid((unsigned)((P + 31) / 32), (unsigned)((S + 31) / 32), (unsigned)K), block(256);
    const unsigned char *l = static_cast<const unsigned char *>(x);
    if (kind == 0)
        hipLaunchKernelGGL((planes_to_rows_kernel<float, float>), grid, block, 0, stream, static_cast<const float *>(x), P, S, K,
                           static_cast<float *>(y));
    else if (kind == 1)
        hipLaunchKernelGGL((planes_to_rows_kernel<unsigned char, unsigned char>), grid, block, 0, stream, l, P, S, K,
                           static_cast<unsigned char *>(y));
    else
        hipLaunchKernelGGL((planes_to_rows_kernel<unsigned char, int>), grid, block, 0, stream, l, P, S, K, static_cast<int *>(y));
    return hipGetLastError();
}

}  // namespace qmri
