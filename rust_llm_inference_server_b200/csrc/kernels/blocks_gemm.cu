// y[M, N] = x[M, K] w[N, K]^T with both operands in e4m3 and a float32 scale for each block of k: x by 128 of a row, w by 128 x 128.
#include "common.cuh"
#include <cuda_fp8.h>

namespace {
constexpr int TB = 64, TK = 32;
__device__ __forceinline__ float code_value(unsigned char c) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3))); }

template <typename OutT>
__global__ __launch_bounds__(256) void blocks_gemm_kernel(const unsigned char* __restrict__ x, long long ldx, const float* __restrict__ sx, const unsigned char* __restrict__ w,
                                                          long long ldw, const float* __restrict__ sw, OutT* __restrict__ y, int M, int N, int K, int k_blocks) {
    pdl_wait();
    __shared__ float xs[TK][TB + 4], ws[TK][TB + 4];
    const int m0 = blockIdx.y * TB, n0 = blockIdx.x * TB, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float acc[4][4] = {};
    for (int kb = 0; kb < k_blocks; ++kb) {
        float part[4][4] = {};
        for (int k0 = kb * 128; k0 < min(kb * 128 + 128, K); k0 += TK) {
            for (int i = threadIdx.x; i < TB * TK; i += 256) {
                const int r = i / TK, c = i % TK;
                xs[c][r] = m0 + r < M && k0 + c < K ? code_value(x[(m0 + r) * ldx + k0 + c]) : 0.f;
                ws[c][r] = n0 + r < N && k0 + c < K ? code_value(w[(n0 + r) * ldw + k0 + c]) : 0.f;
            }
            __syncthreads();
            for (int c = 0; c < TK; ++c)
                for (int i = 0; i < 4; ++i)
                    for (int j = 0; j < 4; ++j) part[i][j] = fmaf(xs[c][ty * 4 + i], ws[c][tx * 4 + j], part[i][j]);
            __syncthreads();
        }
        for (int i = 0; i < 4; ++i) {
            const int m = m0 + ty * 4 + i;
            const float a = m < M ? sx[(long long)kb * M + m] : 0.f;
            for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(part[i][j], a * sw[(long long)(n0 / 128) * k_blocks + kb], acc[i][j]);
        }
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j)
            if (m0 + ty * 4 + i < M && n0 + tx * 4 + j < N) y[(long long)(m0 + ty * 4 + i) * N + n0 + tx * 4 + j] = from_f<OutT>(acc[i][j]);
    pdl_trigger();
}
}  // namespace

// x [M, K] (rows ldx bytes apart), sx [ceil(K / 128), M]; w [N, K] (rows ldw bytes apart), sw [ceil(N / 128), ceil(K / 128)]; y [M, N].
extern "C" int rlis_blocks_gemm(const void* x, long long ldx, const float* sx, const void* w, long long ldw, const float* sw, void* y, int M, int N, int K, int out_dtype,
                                cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0 || (M + TB - 1) / TB > 65535 || (out_dtype != RLIS_F32 && out_dtype != RLIS_BF16)) return RLIS_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)((N + TB - 1) / TB), (unsigned)((M + TB - 1) / TB));
    const unsigned char *xc = static_cast<const unsigned char*>(x), *wc = static_cast<const unsigned char*>(w);
    if (out_dtype == RLIS_F32) rlis_launch(blocks_gemm_kernel<float>, grid, 256, 0, stream, xc, ldx, sx, wc, ldw, sw, (float*)y, M, N, K, (K + 127) / 128);
    else rlis_launch(blocks_gemm_kernel<bf16>, grid, 256, 0, stream, xc, ldx, sx, wc, ldw, sw, (bf16*)y, M, N, K, (K + 127) / 128);
    return RLIS_LAUNCH_CHECK();
}
