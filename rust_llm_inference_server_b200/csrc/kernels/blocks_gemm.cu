// y[M, N] = x[M, K] w[N, K]^T with both operands in e4m3 and a float32 scale for each block of k: x by 128 of a row, w by 128 x 128.
//
//   y[m, n] = sum over blocks b of  sx[b, m] sw[n / 128, b] * (sum over k in b of cx[m, k] cw[n, k])
//
// A block's products are exact in the tensor cores' float32 sums, but two blocks' sums may not meet before they are scaled: a tile's sums of 128 k go to an
// accumulator of their own in tensor memory, and the epilogue's warps take it from there, scale it and add it to the tile's float32 sums, which they keep in
// registers.  So they work beside the tensor core all the time and not after a tile: for each 128 x 128 x 128 products of an SM (256 cycles) they read 16,384 sums
// and add as many, by two in an instruction (fma.rn.f32x2), 64 cycles of the four schedulers.
//
// Many rows (this file): two SMs to a tile of 256 x BN, `tcgen05.mma.cta_group::2` of kind::f8f6f4.  A cluster of two CTAs; CTA r holds rows 128 r .. of x and
// of the result, and half of the tile's rows of w; the instruction, issued by one thread of CTA 0, reads each CTA's x from that CTA's shared memory and w's
// halves from both.  Warp 0 asks for the tiles (bulk tensor copies of 128 k, a row of 128 bytes, 128-byte swizzle; the bytes of both CTAs are counted by CTA
// 0's barrier of the stage); warp 1 of CTA 0 issues the products; `tcgen05.commit` hands the stage back to both producers and the accumulator to both
// epilogues; warps 4-11 are the epilogue, a quarter of the rows and half of the columns each, and tell CTA 0 when they have read an accumulator.
// Few rows: blocks_few.cuh.
//
// Every mbarrier wait is bounded (tcgen05_utils.cuh); a wait that runs out sets the error word, every role runs to its end without further waits, the CTAs
// meet and free their tensor memory.
#include "blocks.cuh"
#include "tcgen05_utils.cuh"

namespace {
using namespace tc;
constexpr int BG_M = 128;                               // rows of a CTA: the pair's tile is twice that
constexpr int BG_A_BYTES = BG_M * QB;
constexpr int BG_THREADS = 384, BG_WARPS = 8;           // three groups of four warps; the last two are the epilogue
// Registers a thread: 168 at launch for every group; the epilogue's 128 sums a thread and two sets of loads want more, the first group gives them up.
constexpr int BG_REGS_LAUNCH = 168, BG_REGS_FIRST = 56, BG_REGS_EPILOGUE = 224;
static_assert(BG_REGS_FIRST + 2 * BG_REGS_EPILOGUE <= 3 * BG_REGS_LAUNCH && BG_THREADS * BG_REGS_LAUNCH <= 65536, "a split above what the launch holds waits for good");
constexpr int BG_TURN = 32 * 128;                       // bytes in which an epilogue warp turns 128 bytes of its 32 rows
constexpr int BG_MAX_STAGES = 8, BG_MAX_BUFFERS = 4;

template <int BN> __host__ __device__ constexpr int bg_stage_bytes() { return BG_A_BYTES + BN / 2 * QB; }
template <int BN> __host__ __device__ constexpr int bg_stages() { return BN == 256 ? 6 : BN == 192 ? 6 : 8; }
template <int BN> __host__ __device__ constexpr int bg_buffers() { return BN == 128 ? 4 : 2; }
template <int BN> constexpr size_t bg_smem() { return (size_t)bg_stages<BN>() * bg_stage_bytes<BN>() + BG_WARPS * BG_TURN + 1024 /* alignment */ + 256; }

struct BgCtrl {
    uint64_t full[BG_MAX_STAGES];           // CTA 0's: both CTAs' bytes of a stage have arrived
    uint64_t empty[BG_MAX_STAGES];          // each CTA's: the products that read the stage are done
    uint64_t acc_full[BG_MAX_BUFFERS];      // each CTA's: a block's sums are complete
    uint64_t acc_empty[BG_MAX_BUFFERS];     // CTA 0's: the sixteen epilogue warps of the pair have read them
    uint32_t tmem_base;
    int abort;
};
static_assert(sizeof(BgCtrl) <= 256, "the control block");

// Instruction descriptor, kind::f8f6f4: float32 accumulator (bits 4-5 = 1), A and B e4m3 (bits 7-9 and 10-12 = 0), both K-major, N / 8 in bits 17-22, M / 16
// in bits 24-28.
__host__ __device__ constexpr uint32_t idesc_e4m3(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }

// A matrix of codes [rows, K] as a 2-D tensor map with boxes of 128 k x box_rows rows, 128-byte swizzle; what lies past K or the rows is read as zeros.
bool make_code_map(CUtensorMap* map, const void* ptr, long long rows, int K, int box_rows, long long row_stride) {
    EncodeTiledFn fn = encode_fn();
    if (fn == nullptr) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)row_stride};
    const cuuint32_t box[2] = {(cuuint32_t)QB, (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

__device__ __forceinline__ uint32_t bg_cta_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// The address of a shared-memory object of CTA `rank` of the cluster, in the cluster's window.
__device__ __forceinline__ uint32_t bg_in_cta(const void* p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
// A tile into this CTA's shared memory; its bytes are counted by the barrier at `bar_cluster_addr`, which may be the other CTA's of the pair.
__device__ __forceinline__ void bg_load_pair(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar_cluster_addr) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(bar_cluster_addr), "r"(x), "r"(y)
                 : "memory");
}
__device__ __forceinline__ void umma_e4m3_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
        "}\n"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// An arrival at the barrier at this offset in both CTAs of the pair once the products issued so far are done.
__device__ __forceinline__ void bg_commit_pair(uint64_t* bar) {
    const unsigned short both = 3;
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(smem_u32(bar)), "h"(both) : "memory");
}
__device__ __forceinline__ void bg_arrive_cluster(uint32_t bar_cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster_addr) : "memory");
}

// Sixteen columns of a lane's row without the wait: the registers may be read only after tmem_ld_wait().
__device__ __forceinline__ void tmem_ld16_nowait(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
// Two sums at once: acc += s * r.
__device__ __forceinline__ void fma2(unsigned long long& acc, uint32_t r0, uint32_t r1, unsigned long long s2) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(r0), "r"(r1));
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(r), "l"(s2));
}
__device__ __forceinline__ unsigned long long twice(float s) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %1};" : "=l"(r) : "r"(__float_as_uint(s)));
    return r;
}
__device__ __forceinline__ float2 two_of(unsigned long long v) {
    uint32_t a, b;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(v));
    return make_float2(__uint_as_float(a), __uint_as_float(b));
}

// 128 bytes of each of a warp's 32 rows (64 bfloat16 or 32 float32 sums of columns col .., a row a lane), by way of shared memory: rows in 16-byte pieces whose
// places are swapped by the row, so that neither side meets in a bank, and an instruction writes the 128 bytes of four rows.
template <typename OutT> constexpr int BG_STORE = 128 / (int)sizeof(OutT);
template <typename OutT>
__device__ __forceinline__ void store_turned(const unsigned long long* acc, uint4* turn, OutT* __restrict__ y, int row0, int col, int M, int end, int N, bool aligned) {
    constexpr int PER = 16 / (int)sizeof(OutT);             // values in a piece
    const int lane = threadIdx.x & 31;
    __syncwarp();
#pragma unroll
    for (int v = 0; v < 8; ++v) {
        uint4 pk;
        if constexpr (sizeof(OutT) == 2) {
            const float2 a = two_of(acc[4 * v]), b = two_of(acc[4 * v + 1]), c = two_of(acc[4 * v + 2]), d = two_of(acc[4 * v + 3]);
            pk = make_uint4(pack_bf16(a.x, a.y), pack_bf16(b.x, b.y), pack_bf16(c.x, c.y), pack_bf16(d.x, d.y));
        } else {
            const float2 a = two_of(acc[2 * v]), b = two_of(acc[2 * v + 1]);
            pk = make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
        }
        turn[lane * 8 + (v ^ (lane & 7))] = pk;
    }
    __syncwarp();
    if (aligned) {
        const int piece = lane & 7, at = col + piece * PER;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int lr = j * 4 + (lane >> 3);
            if (row0 + lr < M && at < end) *reinterpret_cast<uint4*>(y + (size_t)(row0 + lr) * N + at) = turn[lr * 8 + (piece ^ (lr & 7))];
        }
    } else {
        // rows that start anywhere: value by value
        for (int lr = 0; lr < 32 && row0 + lr < M; ++lr)
            for (int c = lane; c < BG_STORE<OutT> && col + c < end; c += 32)
                y[(size_t)(row0 + lr) * N + col + c] = reinterpret_cast<const OutT*>(turn)[(lr * 8 + ((c / PER) ^ (lr & 7))) * PER + c % PER];
    }
}

// Persistent: pair p works on tiles p, p + pairs, ...; tile t -> (n tile t / m_tiles, m tile t % m_tiles), so that the pairs that run together share a few
// rows of w and all of x in L2.
template <int BN, typename OutT>
__global__ __launch_bounds__(BG_THREADS, 1) void blocks_gemm_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                                                                 const float* __restrict__ sx, const float* __restrict__ sw, OutT* __restrict__ y, int M, int N,
                                                                 int k_blocks, int m_tiles, int num_tiles) {
    constexpr int STAGES = bg_stages<BN>(), BUFFERS = bg_buffers<BN>(), B_BYTES = BN / 2 * QB, HALF = BN / 2;
    constexpr uint32_t IDESC = idesc_e4m3(2 * BG_M, BN);
    pdl_wait();
    extern __shared__ unsigned char bg_smem_raw[];
    // the same offset in both CTAs (their dynamic arrays start at the same address): the instruction reads both CTAs' tiles through one descriptor
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(bg_smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char *a_tiles = base, *b_tiles = base + STAGES * BG_A_BYTES, *turns = b_tiles + STAGES * B_BYTES;
    BgCtrl* ctrl = reinterpret_cast<BgCtrl*>(turns + BG_WARPS * BG_TURN);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = bg_cta_rank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        ctrl->abort = 0;
        for (int s = 0; s < STAGES; ++s) {
            bar_init(&ctrl->full[s], 1);
            bar_init(&ctrl->empty[s], 1);
        }
        for (int i = 0; i < BUFFERS; ++i) {
            bar_init(&ctrl->acc_full[i], 1);
            bar_init(&ctrl->acc_empty[i], 2 * BG_WARPS);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {   // one warp of each CTA of the pair: all of tensor memory in both
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctrl->tmem_base)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncwarp();
    cluster_sync_all();         // both CTAs' barriers exist before either is used from the other side
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = ctrl->tmem_base;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(BG_REGS_FIRST));
        if (warp == 0) {
            if (lane == 0) {
                int it = 0;
                for (int tile = pair; tile < num_tiles && !ctrl->abort; tile += pairs) {
                    const int n0 = (tile / m_tiles) * BN, m0 = (tile % m_tiles) * 2 * BG_M;
                    for (int kb = 0; kb < k_blocks; ++kb, ++it) {
                        const int s = it % STAGES;
                        if (it >= STAGES && !bar_wait(&ctrl->empty[s], ((it / STAGES) - 1) & 1, &ctrl->abort)) break;
                        const uint32_t full0 = bg_in_cta(&ctrl->full[s], 0);
                        if (rank == 0) bar_expect_tx(&ctrl->full[s], 2 * (BG_A_BYTES + B_BYTES));
                        bg_load_pair(a_tiles + s * BG_A_BYTES, &map_x, kb * QB, m0 + (int)rank * BG_M, full0);
                        bg_load_pair(b_tiles + s * B_BYTES, &map_w, kb * QB, n0 + (int)rank * HALF, full0);
                    }
                }
            }
        } else if (warp == 1) {
            if (rank == 0) {
                // the whole warp walks the loop and waits, and leaves it together; one lane issues
                int it = 0;
                bool fine = true;
                for (int tile = pair; tile < num_tiles && fine; tile += pairs) {
                    for (int kb = 0; kb < k_blocks; ++kb, ++it) {
                        const int s = it % STAGES, buf = it % BUFFERS;
                        if (it >= BUFFERS && !bar_wait_warp(&ctrl->acc_empty[buf], ((it / BUFFERS) - 1) & 1, &ctrl->abort)) { fine = false; break; }
                        if (!bar_wait_warp(&ctrl->full[s], (it / STAGES) & 1, &ctrl->abort)) { fine = false; break; }
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        if (elect_one()) {
                            const uint64_t adesc = smem_desc_sw128(a_tiles + s * BG_A_BYTES), bdesc = smem_desc_sw128(b_tiles + s * B_BYTES);
    #pragma unroll
                            for (int k = 0; k < QB / 32; ++k)          // 32 codes further along the swizzled row
                                umma_e4m3_pair(tmem_base + (uint32_t)(buf * BN), adesc + (uint64_t)(k * 32 >> 4), bdesc + (uint64_t)(k * 32 >> 4), IDESC, k != 0 ? 1u : 0u);
                            bg_commit_pair(&ctrl->empty[s]);
                            bg_commit_pair(&ctrl->acc_full[buf]);
                        }
                        __syncwarp();
                    }
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(BG_REGS_EPILOGUE));
        // epilogue: warp w may touch TMEM lanes 32 * (w % 4) .. + 31; two warps share them, half of the columns each
        const int q = warp & 3, half = (warp - 4) / 4;
        const int n_blocks = (N + QB - 1) / QB;
        const bool aligned = (N * (int)sizeof(OutT)) % 16 == 0 && (reinterpret_cast<uintptr_t>(y) & 15) == 0;
        uint4* turn = reinterpret_cast<uint4*>(turns + (warp - 4) * BG_TURN);
        int it = 0;
        bool fine = true;
        for (int tile = pair; tile < num_tiles && fine; tile += pairs) {
            const int col0 = (tile / m_tiles) * BN + half * HALF, row0 = (tile % m_tiles) * 2 * BG_M + (int)rank * BG_M + q * 32, row = row0 + lane;
            // this warp's columns lie in one block of w's rows, or (BN 192) in two that meet at a multiple of 32
            const int nb = min(col0 / QB, n_blocks - 1), nb1 = min((col0 + HALF - 1) / QB, n_blocks - 1);
            const int border = BN == 192 ? (col0 / QB + 1) * QB - col0 : HALF;
            const float *pw = sw + (size_t)nb * k_blocks, *pw1 = sw + (size_t)nb1 * k_blocks, *px = sx + min(row, M - 1);
            unsigned long long acc[HALF / 2];
#pragma unroll
            for (int i = 0; i < HALF / 2; ++i) acc[i] = 0ull;
            float a = *px, b = *pw, b1 = BN == 192 ? *pw1 : 0.f;           // the next block's scales are asked for before this one's sums are awaited
            for (int kb = 0; kb < k_blocks; ++kb, ++it) {
                const int buf = it % BUFFERS;
                const unsigned long long s2 = twice(a * b), s2b = BN == 192 ? twice(a * b1) : 0ull;
                if (kb + 1 < k_blocks) {
                    a = px[(size_t)(kb + 1) * M];
                    b = pw[kb + 1];
                    if (BN == 192) b1 = pw1[kb + 1];
                }
                if (!bar_wait_warp(&ctrl->acc_full[buf], (it / BUFFERS) & 1, &ctrl->abort)) { fine = false; break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t from = tmem_base + (uint32_t)(buf * BN + half * HALF) + ((uint32_t)(q * 32) << 16);
                uint32_t r[2][16];
                tmem_ld16_nowait(from, r[0]);
#pragma unroll
                for (int c = 0; c < HALF / 16; ++c) {
                    tmem_ld_wait();
                    if (c + 1 < HALF / 16) tmem_ld16_nowait(from + (uint32_t)((c + 1) * 16), r[(c + 1) & 1]);
                    const unsigned long long s = BN == 192 && c * 16 >= border ? s2b : s2;
#pragma unroll
                    for (int i = 0; i < 8; ++i) fma2(acc[c * 8 + i], r[c & 1][2 * i], r[c & 1][2 * i + 1], s);
                }
                // this warp has read its lanes of the accumulator: CTA 0's product warp may write it again
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) bg_arrive_cluster(bg_in_cta(&ctrl->acc_empty[buf], 0));
            }
            if (!fine) break;
#pragma unroll
            for (int c = 0; c < HALF; c += BG_STORE<OutT>) {
                if constexpr (HALF % BG_STORE<OutT> != 0) {                // bfloat16, 96 columns: 64 and 32
                    if (c + BG_STORE<OutT> > HALF) {
                        unsigned long long rest[BG_STORE<OutT> / 2];
#pragma unroll
                        for (int i = 0; i < BG_STORE<OutT> / 2; ++i) rest[i] = c / 2 + i < HALF / 2 ? acc[(c / 2 + i) % (HALF / 2)] : 0ull;
                        store_turned<OutT>(rest, turn, y, row0, col0 + c, M, min(N, col0 + HALF), N, aligned);
                        continue;
                    }
                }
                store_turned<OutT>(acc + c / 2, turn, y, row0, col0 + c, M, N, N, aligned);
            }
        }
    }
    // nobody leaves, and no tensor memory is freed, while the other CTA may still use this one's
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncwarp();
    cluster_sync_all();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
    }
    pdl_trigger();
}

template <int BN, typename OutT>
int launch_blocks_gemm(const void* x, long long ldx, const float* sx, const void* w, long long ldw, const float* sw, void* y, int M, int N, int K, int sms,
                       cudaStream_t stream) {
    static std::atomic<unsigned long long> allowed{0};
    const cudaError_t e = rlis_allow_smem(blocks_gemm_kernel<BN, OutT>, (int)bg_smem<BN>(), allowed);
    if (e != cudaSuccess) return (int)e;
    CUtensorMap map_x, map_w;
    if (!make_code_map(&map_x, x, M, K, BG_M, ldx) || !make_code_map(&map_w, w, N, K, BN / 2, ldw)) return RLIS_ERR_UNSUPPORTED;
    const int m_tiles = (M + 2 * BG_M - 1) / (2 * BG_M), num_tiles = m_tiles * ((N + BN - 1) / BN), pairs = num_tiles < sms / 2 ? num_tiles : sms / 2;
    rlis_launch_cluster(blocks_gemm_kernel<BN, OutT>, dim3((unsigned)(2 * pairs)), dim3(BG_THREADS), bg_smem<BN>(), stream, dim3(2, 1, 1), map_x, map_w, sx, sw, (OutT*)y,
                        M, N, (K + QB - 1) / QB, m_tiles, num_tiles);
    return RLIS_LAUNCH_CHECK();
}
}  // namespace

// 0 if no bounded wait of these products ever ran out on the current device.
extern "C" int rlis_blocks_gemm_error(void) { return tc::read_error_word(); }
extern "C" int* rlis_blocks_gemm_error_addr(void) { return tc::error_word_addr(); }

// x [M, K] (rows ldx bytes apart), sx [ceil(K / 128), M]; w [N, K] (rows ldw bytes apart), sw [ceil(N / 128), ceil(K / 128)]; y [M, N].  Codes on 16-byte
// boundaries, their rows multiples of 16 bytes apart.
extern "C" int rlis_blocks_gemm(const void* x, long long ldx, const float* sx, const void* w, long long ldw, const float* sw, void* y, int M, int N, int K, int out_dtype,
                                cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0 || (out_dtype != RLIS_F32 && out_dtype != RLIS_BF16) || ldx < K || ldw < K || ldx % 16 != 0 || ldw % 16 != 0 ||
        ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 15) != 0)
        return RLIS_ERR_UNSUPPORTED;
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    // The width of a tile: the one whose rounds over the pairs of SMs come to the fewest columns (a round of narrow tiles is shorter), the widest of equals.
    const long long m_tiles = (M + 2 * BG_M - 1) / (2 * BG_M);
    auto columns = [&](int bn) { const long long tiles = m_tiles * ((N + bn - 1) / bn); return (tiles + sms / 2 - 1) / (sms / 2) * bn; };
    const int bn = columns(256) <= columns(192) && columns(256) <= columns(128) ? 256 : columns(192) <= columns(128) ? 192 : 128;
    const bool f32 = out_dtype == RLIS_F32;
#define RLIS_BG(BN) (f32 ? launch_blocks_gemm<BN, float>(x, ldx, sx, w, ldw, sw, y, M, N, K, sms, stream) : launch_blocks_gemm<BN, bf16>(x, ldx, sx, w, ldw, sw, y, M, N, K, sms, stream))
    return bn == 256 ? RLIS_BG(256) : bn == 192 ? RLIS_BG(192) : RLIS_BG(128);
#undef RLIS_BG
}
