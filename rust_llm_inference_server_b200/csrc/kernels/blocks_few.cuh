// The product of blocks_gemm.cu for few rows: a stream of w from memory, one byte a weight.
//
// The weights are the M side of the instruction: a CTA owns 128 features and a range of the blocks of k; a block of w (128 x 128 codes, 16 KB) arrives by one
// bulk tensor copy into a ring of stages, with the NT x 128 tile of x (NT: rows rounded up to 16, 32, 64 or 128).  Warp 0 asks for the tiles, warp 1 issues
// tcgen05.mma (128 x NT x 32, four a block) into one of several accumulators of NT columns, warps 2-5 take a block's sums from there (a lane a feature, a
// column a row of x), multiply them by sx[row] sw and add them in registers, where a block's products of scales lie in shared memory.
// w has one scale for the CTA's 128 features and a block, so a thread needs no scale of its own.
//
// Matrices with few features would fill few SMs, so k is split over the CTAs of a thread-block cluster (any number up to 16).  Their sums go to shared memory, and
// after a cluster barrier CTA r adds the rows r, r + splits, .. of all CTAs in the order of the splits: the result does not depend on timing.  The number of
// splits depends on N and K alone, so a row has the same bits whatever other rows there are, up to 128.
//
// FUSED (up to 16 rows, not yet in blocks): the CTA puts its part of x into blocks itself, as quantize_rows does, straight into the swizzled layout that the
// instruction reads, while its first tiles of w are on their way; a launch and a round trip of the codes less.
// (Included by blocks_gemm.cu, whose error word it shares.)
#pragma once

namespace {
constexpr int BF_F = 128;                               // features of a CTA
constexpr int BF_THREADS = 192;
constexpr int BF_W_BYTES = BF_F * QB;
constexpr int BF_MAX_STAGES = 6, BF_MAX_BUFFERS = 4, BF_MAX_SPLITS = 16;
constexpr int BF_SCALES = 4096;                         // products of scales that shared memory holds at a time
constexpr int BF_FUSED_BLOCKS = 32;                     // blocks of k up to which a CTA holds its rows of x itself

template <int NT> __host__ __device__ constexpr int bf_stages() { return NT == 16 ? 6 : NT == 32 ? 5 : NT == 64 ? 4 : 3; }
template <int NT> __host__ __device__ constexpr int bf_buffers() { return NT <= 32 ? 4 : 2; }

struct BfCtrl {
    uint64_t full[BF_MAX_STAGES];
    uint64_t empty[BF_MAX_STAGES];
    uint64_t acc_full[BF_MAX_BUFFERS];
    uint64_t acc_empty[BF_MAX_BUFFERS];
    uint32_t tmem_base;
    int abort;
};
static_assert(sizeof(BfCtrl) <= 256, "the control block");

__device__ __forceinline__ void umma_e4m3(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
        "}\n"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// The rows of x that a FUSED launch puts into blocks.
struct PlainRows {
    const void* x;
    long long ld;
    int K;
};

// This CTA's blocks kb0 .. kb1 of x's rows: codes into the tiles [block][16 rows of 128 bytes, 128-byte swizzle], scales times w's into sc [block][16].
template <typename T, bool VEC>
__device__ __forceinline__ void blocks_of_rows(const PlainRows& p, int M, int kb0, int n_kb, const float* __restrict__ sw, unsigned char* tiles, float* sc) {
    constexpr int GROUPS = BF_THREADS / 16, AHEAD = 4;
    const T* x = reinterpret_cast<const T*>(p.x);
    const int group = threadIdx.x >> 4, lane = threadIdx.x & 15, total = M * n_kb;
    for (int first = group; first - group < total; first += GROUPS * AHEAD) {          // (the same number of rounds for all: shuffles are whole warps')
        float v[AHEAD][8];
        int row[AHEAD], kb[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int unit = first + u * GROUPS;
            row[u] = unit < total ? unit / n_kb : -1;
            kb[u] = unit < total ? unit - row[u] * n_kb : 0;
            if (row[u] >= 0) {
                load8<T, VEC>(x + row[u] * p.ld, (kb0 + kb[u]) * QB + lane * 8, p.K, v[u]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[u][i] = 0.f;
            }
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            unsigned amax = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) amax = max(amax, abs_bits(v[u][i]));
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            if (row[u] < 0) continue;
            const Coding c = coding_of(amax);
            unsigned char* to = tiles + kb[u] * (16 * QB) + row[u] * QB + (((lane >> 1) ^ (row[u] & 7)) << 4) + (lane & 1) * 8;
            *reinterpret_cast<uint2*>(to) = make_uint2(codes4(v[u], c), codes4(v[u] + 4, c));
            if (lane == 0) sc[kb[u] * 16 + row[u]] = c.scale * sw[kb0 + kb[u]];
        }
    }
}

template <int NT, int FUSED /* 0: x in blocks; 1: bfloat16 rows, 2: float32; 3, 4: the same in vectors */, typename OutT>
__global__ __launch_bounds__(BF_THREADS) void blocks_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const PlainRows rows,
                                                                const float* __restrict__ sx, const float* __restrict__ sw, OutT* __restrict__ y, int M, int N,
                                                                int k_blocks, int per, int n_stages, int early) {
    static_assert(!FUSED || NT == 16, "rows that a CTA puts into blocks itself are few");
    constexpr int X_BYTES = NT * QB, BUFFERS = bf_buffers<NT>();
    constexpr uint32_t COLS = BUFFERS * NT, IDESC = idesc_e4m3(BF_F, NT);
    extern __shared__ unsigned char bf_smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(bf_smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char *w_tiles = base, *x_tiles = base + n_stages * BF_W_BYTES;         // x: a tile a stage, or (FUSED) a tile a block
    float* sc = reinterpret_cast<float*>(x_tiles + (FUSED ? per : n_stages) * X_BYTES);
    const int chunk = min(per, BF_SCALES / NT);                                       // blocks whose products of scales are held
    BfCtrl* ctrl = reinterpret_cast<BfCtrl*>(sc + chunk * NT);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tile = blockIdx.x, split = blockIdx.y, splits = gridDim.y;
    const int n0 = tile * BF_F, kb0 = split * per, n_kb = min(per, k_blocks - kb0);
    const float* my_sw = sw + (size_t)tile * k_blocks;

    if (threadIdx.x == 0) {
        ctrl->abort = 0;
        for (int s = 0; s < n_stages; ++s) {
            bar_init(&ctrl->full[s], 1);
            bar_init(&ctrl->empty[s], 1);
        }
        for (int i = 0; i < BUFFERS; ++i) {
            bar_init(&ctrl->acc_full[i], 1);
            bar_init(&ctrl->acc_empty[i], 4);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctrl->tmem_base)), "r"(COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = ctrl->tmem_base;

    const int first = min(n_stages, n_kb);
    auto ask_w = [&](int s, int it) {
        bar_expect_tx(&ctrl->full[s], BF_W_BYTES + (FUSED ? 0 : X_BYTES));
        tma_load_2d(w_tiles + s * BF_W_BYTES, &map_w, (kb0 + it) * QB, n0, &ctrl->full[s]);
    };
    if (threadIdx.x == 0 && early)
        for (int it = 0; it < first; ++it) ask_w(it, it);
    pdl_wait();
    if (threadIdx.x == 0 && !early)
        for (int it = 0; it < first; ++it) ask_w(it, it);
    if constexpr (FUSED != 0) {
        __syncwarp();
        if constexpr (FUSED == 1 || FUSED == 3) blocks_of_rows<bf16, FUSED == 3>(rows, M, kb0, n_kb, my_sw, x_tiles, sc);
        else blocks_of_rows<float, FUSED == 4>(rows, M, kb0, n_kb, my_sw, x_tiles, sc);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
    }

    unsigned long long acc[NT / 2];
    bool fine = true;
    if (warp == 0) {
        if (lane == 0) {
            for (int it = 0; it < n_kb; ++it) {
                const int s = it % n_stages;
                if (it >= first) {
                    if (!bar_wait(&ctrl->empty[s], ((it / n_stages) - 1) & 1, &ctrl->abort)) break;
                    ask_w(s, it);
                }
                if (!FUSED) tma_load_2d(x_tiles + s * X_BYTES, &map_x, (kb0 + it) * QB, 0, &ctrl->full[s]);
            }
            pdl_trigger();     // everything this CTA reads is asked for: the next kernel may start its own
        }
    } else if (warp == 1) {
        // the whole warp walks the loop and waits, and leaves it together; one lane issues
        for (int it = 0; it < n_kb; ++it) {
            const int s = it % n_stages, buf = it % BUFFERS;
            if (!bar_wait_warp(&ctrl->full[s], (it / n_stages) & 1, &ctrl->abort)) break;
            if (it >= BUFFERS && !bar_wait_warp(&ctrl->acc_empty[buf], ((it / BUFFERS) - 1) & 1, &ctrl->abort)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint64_t adesc = smem_desc_sw128(w_tiles + s * BF_W_BYTES), bdesc = smem_desc_sw128(x_tiles + (FUSED ? it : s) * X_BYTES);
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < QB / 32; ++k)          // 32 codes further along the swizzled row
                    umma_e4m3(tmem_base + (uint32_t)(buf * NT), adesc + (uint64_t)(k * 32 >> 4), bdesc + (uint64_t)(k * 32 >> 4), IDESC, k != 0 ? 1u : 0u);
                umma_commit(&ctrl->empty[s]);
                umma_commit(&ctrl->acc_full[buf]);
            }
            __syncwarp();
        }
    } else {
        const int q = warp & 3, mine = (warp - 2) * 32 + lane;
#pragma unroll
        for (int i = 0; i < NT / 2; ++i) acc[i] = 0ull;
        for (int it = 0; it < n_kb; ++it) {
            const int at = it % chunk;
            if (!FUSED && at == 0) {
                asm volatile("bar.sync 1, 128;" ::: "memory");         // the last chunk's have been read
                const int n = min(chunk, n_kb - it) * NT;
                for (int i = mine; i < n; i += 128) {
                    const int kb = kb0 + it + i / NT, t = i % NT;
                    sc[i] = t < M ? sx[(size_t)kb * M + t] * my_sw[kb] : 0.f;
                }
                asm volatile("bar.sync 1, 128;" ::: "memory");
            }
            const int buf = it % BUFFERS;
            if (fine) fine = bar_wait_warp(&ctrl->acc_full[buf], (it / BUFFERS) & 1, &ctrl->abort);
            if (!fine) continue;                                         // (to the barriers above, which all four warps meet at)
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t from = tmem_base + (uint32_t)(buf * NT) + ((uint32_t)(q * 32) << 16);
            const ulonglong2* scale = reinterpret_cast<const ulonglong2*>(sc + at * NT);
            constexpr int LW = NT < 32 ? NT : 32;
#pragma unroll
            for (int c = 0; c < NT / LW; ++c) {
                uint32_t r[LW];
                if constexpr (LW == 32) tmem_ld32_pinned(from + (uint32_t)(c * LW), r);
                else tmem_ld16_pinned(from, r);
                if (c + 1 == NT / LW) {
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) bar_arrive(&ctrl->acc_empty[buf]);
                }
#pragma unroll
                for (int i = 0; i < LW / 4; ++i) {
                    const ulonglong2 s = scale[c * (LW / 4) + i];
                    fma2(acc[c * (LW / 2) + 2 * i], r[4 * i], r[4 * i + 1], s.x);
                    fma2(acc[c * (LW / 2) + 2 * i + 1], r[4 * i + 2], r[4 * i + 3], s.y);
                }
            }
        }
    }
    const int f_local = (warp & 3) * 32 + lane, f = n0 + f_local;
    if (splits == 1) {
        if (warp >= 2 && fine && f < N) {
#pragma unroll
            for (int i = 0; i < NT / 2; ++i) {
                const float2 v = two_of(acc[i]);
                if (2 * i < M) y[(size_t)(2 * i) * N + f] = from_f<OutT>(v.x);
                if (2 * i + 1 < M) y[(size_t)(2 * i + 1) * N + f] = from_f<OutT>(v.y);
            }
        }
    } else {
        // the products and copies of this CTA are done, so its stages hold the sums now: [row][feature]
        float* part = reinterpret_cast<float*>(base);
        __syncwarp();
        if (warp >= 2) {
#pragma unroll
            for (int i = 0; i < NT / 2; ++i) {
                const float2 v = two_of(acc[i]);
                if (2 * i < M) part[(2 * i) * BF_F + f_local] = v.x;
                if (2 * i + 1 < M) part[(2 * i + 1) * BF_F + f_local] = v.y;
            }
        }
        cluster_sync_all();
        if (warp >= 2) {
            for (int t = split; t < M; t += splits) {
                float v = 0.f;
#pragma unroll 4
                for (int s = 0; s < splits; ++s) v += ld_dsmem(part + t * BF_F + f_local, (uint32_t)s);
                if (fine && f < N) y[(size_t)t * N + f] = from_f<OutT>(v);
            }
        }
        cluster_sync_all();         // nobody leaves while others read its sums
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(COLS) : "memory");
    }
}

// How a product is cut: CTAs that share a tile's k, and blocks of k for each.
struct FewPlan {
    int tiles, splits, per;
};
FewPlan few_plan(int N, int k_blocks, int sms) {
    FewPlan p;
    p.tiles = (N + BF_F - 1) / BF_F;
    int splits = (2 * sms + p.tiles - 1) / p.tiles;
    if (splits > BF_MAX_SPLITS) splits = BF_MAX_SPLITS;
    if (splits > k_blocks / 2) splits = k_blocks / 2;
    if (splits < 1) splits = 1;
    p.per = (k_blocks + splits - 1) / splits;
    p.splits = (k_blocks + p.per - 1) / p.per;
    return p;
}

template <int NT, int FUSED, typename OutT>
int launch_blocks_few(const PlainRows& rows, const void* x, long long ldx, const float* sx, const void* w, long long ldw, const float* sw, void* y, int M, int N, int K,
                      int early, const FewPlan& p, cudaStream_t stream) {
    CUtensorMap map_w, map_x;
    if (!make_code_map(&map_w, w, N, K, BF_F, ldw)) return RLIS_ERR_UNSUPPORTED;
    map_x = map_w;
    if (!FUSED && !make_code_map(&map_x, x, M, K, NT, ldx)) return RLIS_ERR_UNSUPPORTED;
    int stages = p.per < bf_stages<NT>() ? p.per : bf_stages<NT>();
    // (the stages also hold a CTA's sums for the cluster)
    while (p.splits > 1 && stages * (BF_W_BYTES + (FUSED ? 0 : NT * QB)) < NT * BF_F * 4) ++stages;
    const int chunk = p.per < BF_SCALES / NT ? p.per : BF_SCALES / NT;
    const size_t smem = (size_t)stages * BF_W_BYTES + (size_t)(FUSED ? p.per : stages) * NT * QB + (size_t)chunk * NT * 4 + 1024 /* alignment */ + 256;
    static std::atomic<unsigned long long> allowed{0}, wide{0};
    cudaError_t e = rlis_allow_smem(blocks_few_kernel<NT, FUSED, OutT>, (int)(BF_MAX_STAGES * (BF_W_BYTES + 32 * QB) + BF_FUSED_BLOCKS * 16 * QB + BF_SCALES * 4 + 1280), allowed);
    if (e == cudaSuccess) e = rlis_allow_wide_cluster(blocks_few_kernel<NT, FUSED, OutT>, wide);
    if (e != cudaSuccess) return (int)e;
    rlis_launch_cluster(blocks_few_kernel<NT, FUSED, OutT>, dim3((unsigned)p.tiles, (unsigned)p.splits), BF_THREADS, smem, stream, dim3(1, (unsigned)p.splits, 1), map_w,
                        map_x, rows, sx, sw, (OutT*)y, M, N, (K + QB - 1) / QB, p.per, stages, early);
    return RLIS_LAUNCH_CHECK();
}
}  // namespace
