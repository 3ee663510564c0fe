// Values into e4m3 with a float32 scale for each block (blocks.cuh says how): 128 of a row (activations), or 128 x 128 of a matrix (weights).
// Both kernels read their input once and keep it in registers while the block's largest value is found.  2,048 rows of 14,336 (bfloat16): 15.8 us, 5.6 TB/s, where
// instructions still count beside memory (see blocks.cuh), in float32 27.5 (5.3 TB/s); a matrix of 16,384 x 2,048 33.7 us in float32 (5.0 TB/s), 18.9 in bfloat16; 64 rows
// of 4,096 1.9 us, a launch.
#include "blocks.cuh"

namespace {
// Sixteen lanes take a block of a row, eight values each; a group of lanes takes UNITS blocks, all of whose loads are asked for first.  A block's row is its number
// divided by the blocks of a row: umulhi with ceil(2^32 / blocks) is exact for as many blocks as a launch takes (a division in 64 bits took as many
// instructions as everything else).
constexpr int ROWS_THREADS = 256, UNITS = 4, ROWS_PER_CTA = ROWS_THREADS / 16 * UNITS;
constexpr long long MOST_UNITS = 1 << 16;
template <typename T, bool VEC>
__global__ __launch_bounds__(ROWS_THREADS) void quantize_rows_kernel(const T* __restrict__ x, long long ldx, unsigned char* __restrict__ codes, long long ldc,
                                                                     float* __restrict__ scales, int n_tokens, int rows_per, int K, int k_blocks, unsigned magic) {
    pdl_wait_and_trigger();
    const int group = threadIdx.x >> 4, lane = threadIdx.x & 15;
    const int row0 = blockIdx.y * rows_per, total = min(rows_per, n_tokens - row0) * k_blocks;
    Eight<T> v[UNITS];
    int row[UNITS], kb[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        const int unit = blockIdx.x * ROWS_PER_CTA + u * (ROWS_THREADS / 16) + group;
        const int r = magic != 0u ? (int)__umulhi((unsigned)unit, magic) : unit;
        row[u] = unit < total ? row0 + r : -1;
        kb[u] = unit - r * k_blocks;
        v[u] = row[u] >= 0 ? load8<T, VEC>(x + row[u] * ldx, kb[u] * QB + lane * 8, K) : nothing8<T>();
    }
    // a lane divides for one of the blocks, and the others take it over (all dividing for all: 20.8 us for 18.0 at 2,048 x 14,336)
    unsigned amax[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        amax[u] = amax_bits(v[u]);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) amax[u] = max(amax[u], __shfl_xor_sync(0xffffffffu, amax[u], o));      // within the sixteen lanes
    }
    unsigned own = amax[0];
    int own_row = row[0], own_kb = kb[0];
#pragma unroll
    for (int u = 1; u < UNITS; ++u)
        if (lane == u) own = amax[u], own_row = row[u], own_kb = kb[u];
    const Coding mine = coding_of(own);
    if (lane < UNITS && own_row >= 0) scales[(long long)own_kb * n_tokens + own_row] = mine.scale;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        Coding c;
        c.a = least_of(amax[u]);
        c.factor = __shfl_sync(0xffffffffu, mine.factor, u, 16);
        if (row[u] >= 0) store8<T>(codes + row[u] * ldc, kb[u] * QB + lane * 8, K, v[u], c);
    }
}

// A CTA takes a block of 128 x 128: sixteen lanes a row, 32 rows at a time.
constexpr int MATRIX_THREADS = 512, MATRIX_ROWS = QB / (MATRIX_THREADS / 16);
template <typename T, bool VEC>
__global__ __launch_bounds__(MATRIX_THREADS, sizeof(T) == 4 ? 2 : 3) void quantize_matrix_kernel(const T* __restrict__ w, long long ldw, long long stack_w, unsigned char* __restrict__ codes,
                                                                            long long ldc, float* __restrict__ scales, int N, int K) {
    pdl_wait_and_trigger();
    __shared__ unsigned part[MATRIX_THREADS / 32];
    const int kb = blockIdx.x, nb = blockIdx.y, e = blockIdx.z;
    const int r0 = nb * QB + (threadIdx.x >> 4), k = kb * QB + (threadIdx.x & 15) * 8;
    w += e * stack_w;
    codes += (long long)e * N * ldc;
    Eight<T> v[MATRIX_ROWS];
#pragma unroll
    for (int i = 0; i < MATRIX_ROWS; ++i) {
        const int r = r0 + i * (MATRIX_THREADS / 16);
        v[i] = r < N ? load8<T, VEC>(w + r * ldw, k, K) : nothing8<T>();
    }
    unsigned amax = 0;
#pragma unroll
    for (int i = 0; i < MATRIX_ROWS; ++i) amax = max(amax, amax_bits(v[i]));
    amax = __reduce_max_sync(0xffffffffu, amax);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = amax;
    __syncthreads();
    amax = __reduce_max_sync(0xffffffffu, part[threadIdx.x & (MATRIX_THREADS / 32 - 1)]);
    const Coding c = coding_of(amax);
#pragma unroll
    for (int i = 0; i < MATRIX_ROWS; ++i) {
        const int r = r0 + i * (MATRIX_THREADS / 16);
        if (r < N) store8<T>(codes + r * ldc, k, K, v[i], c);
    }
    if (threadIdx.x == 0) scales[((long long)e * gridDim.y + nb) * gridDim.x + kb] = c.scale;
}

bool in_vectors(const void* p, long long ld, int size) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * size) % 16 == 0; }
}  // namespace

// x [T, K] (rows ldx elements apart) -> codes [T, K] (rows ldc bytes apart, a multiple of 16) and scales float32 [ceil(K / 128), T].
extern "C" int rlis_quantize_rows(const void* x, long long ldx, void* codes, long long ldc, float* scales, int n_tokens, int K, int dtype, cudaStream_t stream) {
    if (n_tokens <= 0 || K <= 0) return 0;
    if ((dtype != RLIS_F32 && dtype != RLIS_BF16) || ldc < ((K + 15) & ~15) || ldc % 16 != 0 || (reinterpret_cast<uintptr_t>(codes) & 15) != 0) return RLIS_ERR_UNSUPPORTED;
    const int k_blocks = (K + QB - 1) / QB;
    // rows in bands whose blocks are few enough for the division by a product
    const int most = MOST_UNITS / k_blocks > 0 ? (int)(MOST_UNITS / k_blocks) : 1, rows_per = n_tokens < most ? n_tokens : most;
    const long long bands = (n_tokens + (long long)rows_per - 1) / rows_per;
    if (k_blocks > MOST_UNITS || bands > 65535) return RLIS_ERR_UNSUPPORTED;
    const unsigned magic = k_blocks > 1 ? (unsigned)(((1ull << 32) + k_blocks - 1) / k_blocks) : 0u;
    const bool vec = in_vectors(x, n_tokens > 1 ? ldx : 0, dtype == RLIS_F32 ? 4 : 2);
    const dim3 grid((unsigned)((rows_per * k_blocks + ROWS_PER_CTA - 1) / ROWS_PER_CTA), (unsigned)bands);
    unsigned char* c = static_cast<unsigned char*>(codes);
    if (dtype == RLIS_F32)
        rlis_launch(vec ? quantize_rows_kernel<float, true> : quantize_rows_kernel<float, false>, grid, ROWS_THREADS, 0, stream, (const float*)x, ldx, c, ldc, scales, n_tokens,
                    rows_per, K, k_blocks, magic);
    else
        rlis_launch(vec ? quantize_rows_kernel<bf16, true> : quantize_rows_kernel<bf16, false>, grid, ROWS_THREADS, 0, stream, (const bf16*)x, ldx, c, ldc, scales, n_tokens,
                    rows_per, K, k_blocks, magic);
    return RLIS_LAUNCH_CHECK();
}

// w [E, N, K] (rows ldw and matrices stack_w elements apart) -> codes [E, N, K] (rows ldc bytes apart) and scales float32 [E, ceil(N / 128), ceil(K / 128)].
extern "C" int rlis_quantize_matrix(const void* w, long long ldw, long long stack_w, void* codes, long long ldc, float* scales, int E, int N, int K, int dtype,
                                    cudaStream_t stream) {
    if (E <= 0 || N <= 0 || K <= 0) return 0;
    const int k_blocks = (K + QB - 1) / QB, n_blocks = (N + QB - 1) / QB;
    if ((dtype != RLIS_F32 && dtype != RLIS_BF16) || ldc < ((K + 15) & ~15) || ldc % 16 != 0 || (reinterpret_cast<uintptr_t>(codes) & 15) != 0 || n_blocks > 65535 || E > 65535)
        return RLIS_ERR_UNSUPPORTED;
    const int size = dtype == RLIS_F32 ? 4 : 2;
    const bool vec = in_vectors(w, N > 1 ? ldw : 0, size) && (E == 1 || (stack_w * size) % 16 == 0);
    const dim3 grid((unsigned)k_blocks, (unsigned)n_blocks, (unsigned)E);
    unsigned char* c = static_cast<unsigned char*>(codes);
    if (dtype == RLIS_F32)
        rlis_launch(vec ? quantize_matrix_kernel<float, true> : quantize_matrix_kernel<float, false>, grid, MATRIX_THREADS, 0, stream, (const float*)w, ldw, stack_w, c, ldc, scales, N, K);
    else
        rlis_launch(vec ? quantize_matrix_kernel<bf16, true> : quantize_matrix_kernel<bf16, false>, grid, MATRIX_THREADS, 0, stream, (const bf16*)w, ldw, stack_w, c, ldc, scales, N, K);
    return RLIS_LAUNCH_CHECK();
}
