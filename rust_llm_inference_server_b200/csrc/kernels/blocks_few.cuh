// The product of blocks_gemm.cu for few rows: a stream of w from memory, one byte a weight.
//
// The weights are the M side of the instruction: a CTA owns 128 features and a range of the blocks of k; a block of w (128 x 128 codes, 16 KB) arrives by one
// bulk tensor copy into a ring of stages, with the NT x 128 tile of x (NT: rows rounded up to 16, 32, 64 or 128).  Warp 0 asks for the tiles, warp 1 issues
// tcgen05.mma (128 x NT x 32, four a block) into one of four accumulators of NT columns, the other warps take a block's sums from there (a lane a feature, a
// column a row of x; groups of four warps share the columns, since the way from a block's sums to the next is a chain of waits, as long as a block of w takes
// to arrive), multiply them by sx[row] sw and add them in registers.  w has one scale for the CTA's 128 features and a block; the products of scales lie in
// shared memory.
//
// Matrices with few features would fill few SMs, so k is split over the CTAs of a thread-block cluster (any number up to 16).  Their sums go to shared memory, and
// after a cluster barrier CTA r adds the rows r, r + splits, .. of all CTAs in the order of the splits: the result does not depend on timing.  The number of
// splits depends on N and K alone up to 64 rows (few_splits), so a row has the same bits whatever other rows there are.
// 8 rows x 16,384 of K 2048 from rows in blocks 8.4 us (4.0 TB/s; plain rows, put into blocks by the product, 10.3), 64 x 4,096 of K 14336
// 16.0, one row x 2,048 of K 2048, over weights that no cache holds, 4.1 (plain or not): a launch, the first tiles' way from memory and the cluster's meeting before
// anything else.
// (Included by blocks_gemm.cu, whose error word it shares.)
#pragma once

namespace {
constexpr int BF_F = 128;                               // features of a CTA
constexpr int BF_W_BYTES = BF_F * QB;
constexpr int BF_MAX_STAGES = 6, BF_BUFFERS = 4, BF_MAX_SPLITS = 16;
constexpr int BF_SCALES = 4096;                         // products of scales that shared memory holds at a time

template <int NT> __host__ __device__ constexpr int bf_groups() { return NT == 128 ? 4 : NT == 16 ? 1 : 2; }      // of four warps, NT / groups columns each
template <int NT> __host__ __device__ constexpr int bf_threads() { return 64 + 128 * bf_groups<NT>(); }
template <int NT> __host__ __device__ constexpr int bf_ctas() { return NT == 128 ? 1 : 2; }                       // that fit an SM

struct BfCtrl {
    uint64_t full[BF_MAX_STAGES];
    uint64_t empty[BF_MAX_STAGES];
    uint64_t acc_full[BF_BUFFERS];
    uint64_t acc_empty[BF_BUFFERS];
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

// Plain rows of x, put into blocks here: by every CTA those of its range of k, whose codes lie in shared memory as the bulk copies would leave them.  `vec`: 16-byte
// loads.
template <typename T> struct PlainRows {
    const T* x;
    long long ldx;
    int K, vec;
};
struct NoRows {};
template <typename Rows> struct PlainValueOf;
template <typename T> struct PlainValueOf<PlainRows<T>> { using type = T; };
template <typename Rows> using PlainValue = typename PlainValueOf<Rows>::type;

// Warps that put rows into blocks: the takers and others, which have nothing else to do.  Sixteen lanes a block of a row, up to four of them at a time.
constexpr int PLAIN_MOST_WARPS = 16, PLAIN_AT_ONCE = 4;

template <int NT, typename OutT, typename Rows /* NoRows: codes by map_x and sx */>
__global__ __launch_bounds__(std::is_same<Rows, NoRows>::value ? bf_threads<NT>() : 64 + 32 * PLAIN_MOST_WARPS, std::is_same<Rows, NoRows>::value ? bf_ctas<NT>() : 1)
void blocks_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                                                                                     const Rows rows, const float* __restrict__ sx, const float* __restrict__ sw,
                                                                                     OutT* __restrict__ y, int M, int N, int k_blocks, int per, int n_stages, int early) {
    constexpr bool PLAIN = !std::is_same<Rows, NoRows>::value;
    constexpr int X_BYTES = NT * QB, GROUPS = bf_groups<NT>(), C = NT / GROUPS, TAKERS = 128 * GROUPS;
    constexpr uint32_t COLS = BF_BUFFERS * NT, IDESC = idesc_e4m3(BF_F, NT);
    extern __shared__ unsigned char bf_smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(bf_smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char *w_tiles = base, *x_tiles = base + n_stages * BF_W_BYTES;
    float* sc = reinterpret_cast<float*>(x_tiles + (PLAIN ? per : n_stages) * X_BYTES);
    const int chunk = min(per, BF_SCALES / NT);                                       // blocks whose products of scales are held
    BfCtrl* ctrl = reinterpret_cast<BfCtrl*>(sc + chunk * NT);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tile = blockIdx.x, split = blockIdx.y, splits = gridDim.y;
    const int n0 = tile * BF_F, kb0 = split * per, n_kb = min(per, k_blocks - kb0);
    const float* my_sw = sw + (size_t)tile * k_blocks;
    const bool taker = warp >= 2 && (!PLAIN || warp < 2 + 4 * GROUPS);

    if (threadIdx.x == 0) {
        ctrl->abort = 0;
        for (int s = 0; s < n_stages; ++s) {
            bar_init(&ctrl->full[s], 1);
            bar_init(&ctrl->empty[s], 1);
        }
        for (int i = 0; i < BF_BUFFERS; ++i) {
            bar_init(&ctrl->acc_full[i], 1);
            bar_init(&ctrl->acc_empty[i], 4 * GROUPS);
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
        bar_expect_tx(&ctrl->full[s], BF_W_BYTES + (PLAIN ? 0 : X_BYTES));
        tma_load_2d(w_tiles + s * BF_W_BYTES, &map_w, (kb0 + it) * QB, n0, &ctrl->full[s]);
    };
    // (128-byte rows of zeros where x has no row; every wait below that fails ends its loop, so that all threads come to the barriers at the end)
    unsigned long long acc[C / 2];
    bool fine = true;
    if (warp == 0) {
        if (lane == 0) {
            if (early)
                for (int it = 0; it < first; ++it) ask_w(it, it);
            pdl_wait();
            for (int it = 0, s = 0, phase = 1; it < n_kb; ++it) {
                if (it >= first && !bar_wait(&ctrl->empty[s], phase, &ctrl->abort)) break;
                if (it >= first || !early) ask_w(s, it);
                if constexpr (!PLAIN) tma_load_2d(x_tiles + s * X_BYTES, &map_x, (kb0 + it) * QB, 0, &ctrl->full[s]);
                if (++s == n_stages) s = 0, phase ^= 1;
            }
            pdl_trigger();     // everything this CTA reads is asked for: the next kernel may start its own
        }
    } else if (warp == 1) {
        if constexpr (PLAIN) asm volatile("bar.sync 2, %0;" ::"r"((int)blockDim.x - 32) : "memory");           // x's codes are there
        // the whole warp walks the loop and waits, and leaves it together; one lane issues
        for (int it = 0, s = 0, phase = 0; it < n_kb; ++it) {
            const int buf = it % BF_BUFFERS;
            if (!bar_wait_warp(&ctrl->full[s], phase, &ctrl->abort)) break;
            const uint64_t adesc = smem_desc_sw128(w_tiles + s * BF_W_BYTES), bdesc = smem_desc_sw128(x_tiles + (PLAIN ? it : s) * X_BYTES);
            if (it >= BF_BUFFERS && !bar_wait_warp(&ctrl->acc_empty[buf], ((it / BF_BUFFERS) - 1) & 1, &ctrl->abort)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < QB / 32; ++k)          // 32 codes further along the swizzled row
                    umma_e4m3(tmem_base + (uint32_t)(buf * NT), adesc + (uint64_t)(k * 32 >> 4), bdesc + (uint64_t)(k * 32 >> 4), IDESC, k != 0 ? 1u : 0u);
                umma_commit(&ctrl->empty[s]);
                umma_commit(&ctrl->acc_full[buf]);
            }
            __syncwarp();
            if (++s == n_stages) s = 0, phase ^= 1;
        }
    } else {
        pdl_wait();
        const int q = warp & 3, group = (warp - 2) / 4, mine = (int)threadIdx.x - 64;
#pragma unroll
        for (int i = 0; i < C / 2; ++i) acc[i] = 0ull;
        if constexpr (PLAIN) {
            using T = PlainValue<Rows>;
            const int l16 = mine & 15, units = M * n_kb, step = ((int)blockDim.x - 64) / 16;
            Eight<T> v[PLAIN_AT_ONCE];
            int t[PLAIN_AT_ONCE], b[PLAIN_AT_ONCE];
#pragma unroll
            for (int i = 0; i < PLAIN_AT_ONCE; ++i) {
                const int unit = (mine >> 4) + i * step;
                b[i] = unit / M;
                t[i] = unit < units ? unit - b[i] * M : -1;
                const T* row = rows.x + t[i] * rows.ldx;
                const int k = (kb0 + b[i]) * QB + l16 * 8;
                v[i] = t[i] < 0 ? nothing8<T>() : rows.vec ? load8<T, true>(row, k, rows.K) : load8<T, false>(row, k, rows.K);
            }
#pragma unroll
            for (int i = 0; i < PLAIN_AT_ONCE; ++i) {
                if (i * step >= units) break;
                unsigned amax = amax_bits(v[i]);
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                if (t[i] < 0) continue;
                const Coding c = coding_of(amax);
                *reinterpret_cast<uint2*>(x_tiles + b[i] * X_BYTES + t[i] * QB + ((l16 >> 1) ^ (t[i] & 7)) * 16 + (l16 & 1) * 8) = codes8<T>(v[i], c);
                if (l16 == 0) sc[b[i] * NT + t[i]] = c.scale * my_sw[kb0 + b[i]];
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            asm volatile("bar.sync 2, %0;" ::"r"((int)blockDim.x - 32) : "memory");
        }
        for (int it0 = 0; it0 < n_kb && taker; it0 += chunk) {
            const int n = min(chunk, n_kb - it0);
            if constexpr (!PLAIN) {
                asm volatile("bar.sync 1, %0;" ::"n"(TAKERS) : "memory");         // the last chunk's have been read
                for (int i = mine; i < n * NT; i += TAKERS) {
                    const int kb = kb0 + it0 + i / NT, t = i % NT;
                    sc[i] = t < M ? sx[(size_t)kb * M + t] * my_sw[kb] : 0.f;
                }
                asm volatile("bar.sync 1, %0;" ::"n"(TAKERS) : "memory");
            }
            const ulonglong2* scale = reinterpret_cast<const ulonglong2*>(sc + group * C);
            for (int i = 0; i < n && fine; ++i, scale += NT / 4) {
                const int it = it0 + i, buf = it % BF_BUFFERS;
                fine = bar_wait_warp(&ctrl->acc_full[buf], (it / BF_BUFFERS) & 1, &ctrl->abort);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t from = tmem_base + (uint32_t)(buf * NT + group * C) + ((uint32_t)(q * 32) << 16);
                uint32_t r[C];
                if constexpr (C == 32) tmem_ld32_pinned(from, r);
                else tmem_ld16_pinned(from, r);
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) bar_arrive(&ctrl->acc_empty[buf]);
#pragma unroll
                for (int j = 0; j < C / 4; ++j) {
                    const ulonglong2 s2 = scale[j];
                    fma2(acc[2 * j], r[4 * j], r[4 * j + 1], s2.x);
                    fma2(acc[2 * j + 1], r[4 * j + 2], r[4 * j + 3], s2.y);
                }
            }
        }
    }
    // The sums are in registers: tensor memory goes back before the cluster meets.  A CTA that held it there would wait for CTAs that may wait for tensor memory, which
    // another kernel's CTAs hold that wait for their own cluster in turn; so whoever holds some here waits for nothing but its own copies and products.
    // (The takers only say that they have read theirs, and the warp that gives it back has arrived at the cluster's barrier before: 0.2 to 0.3 us less than a barrier of all.)
    __syncwarp();
    if (warp == 1) {
        if (splits > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("bar.sync 3, %0;" ::"n"(TAKERS + 32) : "memory");
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(COLS) : "memory");
    } else if (taker) {
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        asm volatile("bar.arrive 3, %0;" ::"n"(TAKERS + 32) : "memory");
    }
    const int f_local = (warp & 3) * 32 + lane, f = n0 + f_local, group = (warp - 2) / 4, t0 = group * C;
    if (splits == 1) {
        if (taker && fine && f < N) {
#pragma unroll
            for (int i = 0; i < C / 2; ++i) {
                const float2 v = two_of(acc[i]);
                if (t0 + 2 * i < M) y[(size_t)(t0 + 2 * i) * N + f] = from_f<OutT>(v.x);
                if (t0 + 2 * i + 1 < M) y[(size_t)(t0 + 2 * i + 1) * N + f] = from_f<OutT>(v.y);
            }
        }
    } else {
        // the products and copies of this CTA are done, so its stages hold the sums now: [row][feature]
        float* part = reinterpret_cast<float*>(base);
        if (taker) {
#pragma unroll
            for (int i = 0; i < C / 2; ++i) {
                const float2 v = two_of(acc[i]);
                if (t0 + 2 * i < M) part[(t0 + 2 * i) * BF_F + f_local] = v.x;
                if (t0 + 2 * i + 1 < M) part[(t0 + 2 * i + 1) * BF_F + f_local] = v.y;
            }
        }
        if (warp == 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        else cluster_sync_all();
        if (taker) {
            for (int t = split + group * splits; t < M; t += GROUPS * splits) {
                float v = 0.f;
#pragma unroll 4
                for (int s = 0; s < splits; ++s) v += ld_dsmem(part + t * BF_F + f_local, (uint32_t)s);
                if (fine && f < N) y[(size_t)t * N + f] = from_f<OutT>(v);
            }
        }
        cluster_sync_all();         // nobody leaves while others read its sums
    }
}

// CTAs that share a tile's k: a power of two (such clusters leave no SMs of a group of them idle), the smallest that gives work to three quarters of the SMs.  A CTA
// streams a block in 0.4 us at the fastest, so fewer leave memory idle; more share the same stream, and one that finds no place costs a second round.  8 rows, us:
// 4,096 of K 14336 (32 tiles) in 2, 4, 8, 9 splits 19.9, 12.8, 12.7, 13.0 (a cluster of 9 too many: 18.3); 6,144 of K 4096 (48) in 2, 4, 6, 8 8.8, 7.8, 12.6, 7.8;
// 16,384 of K 2048 (128) in 1, 2, 3 8.3, 9.1, 9.3 to 15.1.  With 128 rows a CTA fills an SM, and clusters of more than 4 find too few places.
template <int NT> int few_splits(int tiles, int k_blocks, int sms) {
    int s = 1;
    if (NT == 128)
        while (s < 4 && 2 * s * tiles * 10 <= 9 * sms) s *= 2;
    else
        while (s < BF_MAX_SPLITS && 4 * s * tiles < 3 * sms) s *= 2;
    const int most = k_blocks / 2;
    return s < most ? s : most < 1 ? 1 : most;
}
// Stages of the ring: six for a CTA that has an SM to itself, which clusters of four find for nine tenths of the SMs (64 x 4,096 of K 14336, 128 CTAs: 15.9 us for 16.6 with
// four, plain rows 19.7 for 24.2, since two CTAs on an SM while others wait for the launch before is what four allow); four so that two CTAs fit, for larger clusters and
// where there are more CTAs than SMs; and as few as keep tensor memory enough for many CTAs an SM where there are several for each (128,256 features of K 2048: 40.2, 41.4
// and 45.2 us with 2, 4 and 6).
template <int NT> int few_stages(int tiles, int splits, int sms) {
    if (NT == 128 || (splits == 1 && tiles <= sms) || (splits > 1 && splits <= 4 && 10 * tiles * splits <= 9 * sms)) return 6;
    return splits > 1 || tiles <= 4 * sms || NT == 64 ? 4 : NT == 16 ? 2 : 3;
}

// The splits, the blocks of a split and the stages of a product.
struct FewPlan {
    int tiles, k_blocks, splits, per, stages, chunk;
};
template <int NT> FewPlan few_plan(int N, int K, int sms) {
    FewPlan f;
    f.tiles = (N + BF_F - 1) / BF_F, f.k_blocks = (K + QB - 1) / QB;
    f.splits = few_splits<NT>(f.tiles, f.k_blocks, sms);
    f.per = (f.k_blocks + f.splits - 1) / f.splits;
    f.splits = (f.k_blocks + f.per - 1) / f.per;
    f.stages = few_stages<NT>(f.tiles, f.splits, sms);
    if (f.stages > f.per) f.stages = f.per;
    while (f.splits > 1 && f.stages * (BF_W_BYTES + NT * QB) < NT * BF_F * 4) ++f.stages;         // (they also hold a CTA's sums for the cluster)
    f.chunk = f.per < BF_SCALES / NT ? f.per : BF_SCALES / NT;
    return f;
}
template <int NT, typename OutT>
int launch_blocks_few(const void* x, long long ldx, const float* sx, const void* w, long long ldw, const float* sw, void* y, int M, int N, int K, int early, int sms,
                      cudaStream_t stream) {
    static std::atomic<unsigned long long> allowed{0}, wide{0};
    constexpr int STAGE_BYTES = BF_W_BYTES + NT * QB;
    cudaError_t e = rlis_allow_smem(blocks_few_kernel<NT, OutT, NoRows>, BF_MAX_STAGES * STAGE_BYTES + BF_SCALES * 4 + 1280, allowed);
    if (e == cudaSuccess) e = rlis_allow_wide_cluster(blocks_few_kernel<NT, OutT, NoRows>, wide);
    if (e != cudaSuccess) return (int)e;
    CUtensorMap map_w, map_x;
    if (!make_code_map(&map_w, w, N, K, BF_F, ldw) || !make_code_map(&map_x, x, M, K, NT, ldx)) return RLIS_ERR_UNSUPPORTED;
    const FewPlan f = few_plan<NT>(N, K, sms);
    rlis_launch_cluster(blocks_few_kernel<NT, OutT, NoRows>, dim3((unsigned)f.tiles, (unsigned)f.splits), bf_threads<NT>(),
                        (size_t)f.stages * STAGE_BYTES + (size_t)f.chunk * NT * 4 + 1280, stream, dim3(1, (unsigned)f.splits, 1), map_w, map_x, NoRows{}, sx, sw, (OutT*)y, M, N,
                        f.k_blocks, f.per, f.stages, early);
    return RLIS_LAUNCH_CHECK();
}

constexpr int PLAIN_NT = 16;            // rows up to which they may be put into blocks by the product
constexpr int PLAIN_SMEM = 227 * 1024, PLAIN_TWICE = 113 * 1024;        // of an SM; of which two CTAs fit one
int plain_smem(const FewPlan& f) { return f.stages * BF_W_BYTES + f.per * PLAIN_NT * (QB + 4) + 1280; }
// A CTA that has an SM to itself takes sixteen warps; clusters want two CTAs on an SM to find their places.
int plain_warps(const FewPlan& f, int sms) { return f.splits == 1 && f.tiles <= sms ? PLAIN_MOST_WARPS : PLAIN_MOST_WARPS / 2; }
// Whether the product puts plain rows into blocks itself: where a CTA's warps do so in one go (more take longer than a launch before, which does it once for all CTAs),
// and in a round of CTAs.  One launch / two, us: 1 x 2,048 of K 2048 3.9 / 4.9, 16 x 2,048 5.2 / 6.4, 1 x 16,384 8.6 / 10.0, 8 x 16,384 10.3 / 10.8, 2 x 4,096 of
// K 14336 15.0 / 15.5; beyond it (in several goes) 8 x 37,000 of K 2048 18.0 / 16.1, 4 x 4,096 of K 14336 16.7 / 15.6, 1 x 28,672 of K 4096 28.7 / 22.0.
// A call of one launch takes the host 9 us for 13.
bool plain_rows_fit(int M, int N, int K, int sms) {
    if (M > PLAIN_NT) return false;
    const FewPlan f = few_plan<PLAIN_NT>(N, K, sms);
    const int smem = plain_smem(f);
    return M * f.per <= 2 * PLAIN_AT_ONCE * plain_warps(f, sms) && smem <= PLAIN_SMEM && f.tiles * f.splits <= (smem <= PLAIN_TWICE ? 2 * sms : sms);
}
template <typename T, typename OutT>
int launch_blocks_few_plain(const void* x, long long ldx, const void* w, long long ldw, const float* sw, void* y, int M, int N, int K, int early, int sms, cudaStream_t stream) {
    static std::atomic<unsigned long long> allowed{0}, wide{0};
    constexpr int NT = PLAIN_NT;
    using Rows = PlainRows<T>;
    cudaError_t e = rlis_allow_smem(blocks_few_kernel<NT, OutT, Rows>, PLAIN_SMEM, allowed);
    if (e == cudaSuccess) e = rlis_allow_wide_cluster(blocks_few_kernel<NT, OutT, Rows>, wide);
    if (e != cudaSuccess) return (int)e;
    CUtensorMap map_w;
    if (!make_code_map(&map_w, w, N, K, BF_F, ldw)) return RLIS_ERR_UNSUPPORTED;
    const FewPlan f = few_plan<NT>(N, K, sms);
    const int vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (M == 1 || (ldx * (long long)sizeof(T)) % 16 == 0) ? 1 : 0;
    rlis_launch_cluster(blocks_few_kernel<NT, OutT, Rows>, dim3((unsigned)f.tiles, (unsigned)f.splits), 64 + 32 * plain_warps(f, sms),
                        (size_t)plain_smem(f), stream, dim3(1, (unsigned)f.splits, 1), map_w, map_w,
                        Rows{static_cast<const T*>(x), ldx, K, vec}, (const float*)nullptr, sw, (OutT*)y, M, N, f.k_blocks, f.per, f.stages, early);
    return RLIS_LAUNCH_CHECK();
}
}  // namespace
