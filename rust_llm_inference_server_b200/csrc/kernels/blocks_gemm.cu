// y[M, N] = x[M, K] w[N, K]^T with both operands in e4m3 and a float32 scale for each block of k: x by 128 of a row, w by 128 x 128.
//
//   y[m, n] = sum over blocks b of  sx[b, m] sw[n / 128, b] * (sum over k in b of cx[m, k] cw[n, k])
//
// Two codes' product is exact and a block's sum of them float32 (they reach over more than its 24 bits: the instruction of each 32 k may cut a unit off it), but two blocks'
// sums may not meet before they are scaled: a tile's sums of 128 k go to an accumulator of their own in tensor memory, and the epilogue's warps take it from there,
// scale it and add it to the tile's float32 sums, which they keep in registers.  So they work beside the tensor core all the time and not after a tile: for each 128 x 128 x 128 products of an SM (256 cycles) they read 16,384 sums
// and add as many, by two in an instruction (fma.rn.f32x2), 64 cycles of the four schedulers.
//
// Many rows (this file): two SMs to a tile of 256 x BN, `tcgen05.mma.cta_group::2` of kind::f8f6f4.  A cluster of two CTAs; CTA r holds rows 128 r .. of x and
// of the result, and half of the tile's rows of w; the instruction, issued by one thread of CTA 0, reads each CTA's x from that CTA's shared memory and w's
// halves from both.  Warp 0 asks for the tiles (bulk tensor copies of 128 k, a row of 128 bytes, 128-byte swizzle; the bytes of both CTAs are counted by CTA
// 0's barrier of the stage); warp 1 of CTA 0 issues the products; `tcgen05.commit` hands the stage back to both producers and the accumulator to both
// epilogues; warps 4-11 are the epilogue, a quarter of the rows and half of the columns each, and tell CTA 0 when they have read an accumulator.
// Few rows: blocks_few.cuh.
//
// What bounds it (2,048 x 16,384 of K 2048, 63 to 64 us, 2,160 TFLOP/s; the nominal e4m3 rate would be 31): the tiles' way from the second-level cache (what is left without
// products and sums takes 44 us, in tiles of 128 columns 73, 11 TB/s), the epilogue's sums (55 without them) and the products (55 with a quarter of them) are of one
// size, and none hides the others whole.  (The hand-over of an accumulator by an arrive that releases waited for the loads of scales on their way, 1,050 to 1,300
// cycles a block: 132 us; the widths of loads from tensor memory make no difference.)
//
// Every mbarrier wait is bounded (tcgen05_utils.cuh); a wait that runs out sets the error word, every role runs to its end without further waits, the CTAs
// meet and free their tensor memory.  The allocation of tensor memory and the cluster's barriers have no bound, so no CTA may hold the one while it waits for the other beside
// a kernel that does the same.  Here the launch takes the registers of a whole SM, and no other CTA that has tensor memory fits beside it; blocks_few.cuh gives its back
// before its cluster meets.
#include "blocks.cuh"
#include "tcgen05_utils.cuh"
#include <algorithm>

namespace {
using namespace tc;
constexpr int BG_M = 128;                               // rows of a CTA: the pair's tile is twice that
constexpr int BG_A_BYTES = BG_M * QB;
constexpr int BG_THREADS = 384, BG_WARPS = 8;           // three groups of four warps; the last two are the epilogue
// Registers a thread: 168 at launch for every group; the epilogue's 128 sums a thread and two sets of loads want more, the first group gives them up.
constexpr int BG_REGS_LAUNCH = 168, BG_REGS_FIRST = 56, BG_REGS_EPILOGUE = 224;
static_assert(BG_REGS_FIRST + 2 * BG_REGS_EPILOGUE <= 3 * BG_REGS_LAUNCH && BG_THREADS * BG_REGS_LAUNCH <= 65536, "a split above what the launch holds waits for good");
static_assert(65536 - BG_THREADS * BG_REGS_LAUNCH < 4 * 32 * 16, "a CTA that holds tensor memory has four warps at least, of sixteen registers and more a thread");
constexpr int BG_MAX_STAGES = 6, BG_MAX_BUFFERS = 4;
constexpr int BG_MAX_SPLITS = 3;                        // the first pair's stages hold the others' sums
constexpr int BG_STAGING = 8192;                        // bytes of results that an epilogue warp keeps for its stores at most

template <int BN> __host__ __device__ constexpr int bg_stage_bytes() { return BG_A_BYTES + BN / 2 * QB; }
template <int BN> __host__ __device__ constexpr int bg_stages() { return BN == 128 ? 6 : 5; }
static_assert((BG_MAX_SPLITS - 1) * 128 * BG_M * 4 <= bg_stages<128>() * bg_stage_bytes<128>(), "room for the other pairs' sums");
template <int BN> __host__ __device__ constexpr int bg_buffers() { return BN == 128 ? 4 : 2; }
// Columns that one store takes: 128 bytes of a row.
template <typename OutT> __host__ __device__ constexpr int bg_store_cols() { return 128 / (int)sizeof(OutT); }
template <int BN, typename OutT> __host__ __device__ constexpr int bg_staging() {
    return BN / 2 * 32 * (int)sizeof(OutT) < BG_STAGING ? BN / 2 * 32 * (int)sizeof(OutT) : BG_STAGING;
}
template <int BN, typename OutT> constexpr size_t bg_smem() {
    return (size_t)bg_stages<BN>() * bg_stage_bytes<BN>() + BG_WARPS * bg_staging<BN, OutT>() + 1024 /* alignment */ + 256;
}

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
__device__ __forceinline__ void bg_commit_pair(uint64_t* bar, uint32_t leader) {
    const unsigned short both = (unsigned short)(3u << leader);
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(smem_u32(bar)), "h"(both) : "memory");
}
// (Relaxed: what it hands over is tensor memory, whose loads have been waited for and fenced; a release would also wait for the next block's scales, which are on
// their way from memory: 1,050 to 1,300 cycles a block.)
__device__ __forceinline__ void bg_arrive_cluster(uint32_t bar_cluster_addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster_addr) : "memory");
}

// 32 columns of a lane's row; the registers pass through the statements behind the wait, so that nothing that reads them is moved ahead of it.
__device__ __forceinline__ void tmem_ld32_pinned(uint32_t taddr, uint32_t (&r)[32]) {
    tmem_ld32(taddr, r);
#pragma unroll
    for (int i = 0; i < 32; i += 8)
        asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]));
}
__device__ __forceinline__ void tmem_ld16_pinned(uint32_t taddr, uint32_t (&r)[16]) {
    tmem_ld16(taddr, r);
#pragma unroll
    for (int i = 0; i < 16; i += 8)
        asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]));
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
__device__ __forceinline__ void add2(unsigned long long& acc, float a, float b) {
    unsigned long long v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(__float_as_uint(a)), "r"(__float_as_uint(b)));
    asm("add.rn.f32x2 %0, %0, %1;" : "+l"(acc) : "l"(v));
}
__device__ __forceinline__ float2 two_of(unsigned long long v) {
    uint32_t a, b;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(v));
    return make_float2(__uint_as_float(a), __uint_as_float(b));
}

// COLS sums (128 bytes) of each of a warp's 32 rows (a row a lane) on their way out, in the layout that a bulk tensor copy of 32 rows reads: 16-byte pieces, piece c of
// row r at c ^ (r % 8), so that a quarter of a warp's lanes meet in no bank.
__device__ __forceinline__ int staged_piece(int row, int piece) { return row * 8 + (piece ^ (row & 7)); }
template <int COLS, typename OutT>
__device__ __forceinline__ void stage_sums(const unsigned long long* acc, uint4* to) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int v = 0; v < COLS * (int)sizeof(OutT) / 16; ++v) {
        uint4 pk;
        if constexpr (sizeof(OutT) == 2) {
            const float2 a = two_of(acc[4 * v]), b = two_of(acc[4 * v + 1]), c = two_of(acc[4 * v + 2]), d = two_of(acc[4 * v + 3]);
            pk = make_uint4(pack_bf16(a.x, a.y), pack_bf16(b.x, b.y), pack_bf16(c.x, c.y), pack_bf16(d.x, d.y));
        } else {
            const float2 a = two_of(acc[2 * v]), b = two_of(acc[2 * v + 1]);
            pk = make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
        }
        to[staged_piece(lane, v)] = pk;
    }
}
// The same for results whose rows start anywhere: value by value.
template <int COLS, typename OutT>
__device__ __forceinline__ void store_staged(const uint4* from, OutT* __restrict__ y, int row0, int col, int M, int N) {
    constexpr int PER = 16 / (int)sizeof(OutT);
    const int lane = threadIdx.x & 31;
    for (int r = 0; r < 32 && row0 + r < M; ++r)
#pragma unroll
        for (int c = lane; c < COLS; c += 32)
            if (col + c < N) y[(size_t)(row0 + r) * N + col + c] = reinterpret_cast<const OutT*>(from)[staged_piece(r, c / PER) * PER + c % PER];
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(smem_u32(src)), "r"(x), "r"(y) : "memory");
}

// Persistent: pair p works on tiles p, p + pairs, ...; tile t -> (n tile t / m_tiles, m tile t % m_tiles), so that the pairs that run together share a few
// rows of w and all of x in L2.  With few tiles the pairs of a cluster share one tile's k instead (splits of them, a tile a cluster): the others hand their sums to
// the first through its shared memory, which adds them in the order of the splits.
template <int BN, typename OutT>
__global__ __launch_bounds__(BG_THREADS, 1) void blocks_gemm_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                                                                    const __grid_constant__ CUtensorMap map_y, const float* __restrict__ sx,
                                                                    const float* __restrict__ sw, OutT* __restrict__ y, int M, int N, int k_blocks, int per, int m_tiles,
                                                                    int num_tiles, int splits, int bulk_stores, int early) {
    constexpr int STAGES = bg_stages<BN>(), BUFFERS = bg_buffers<BN>(), B_BYTES = BN / 2 * QB, HALF = BN / 2;
    constexpr uint32_t IDESC = idesc_e4m3(2 * BG_M, BN);
    extern __shared__ unsigned char bg_smem_raw[];
    // the same offset in both CTAs (their dynamic arrays start at the same address): the instruction reads both CTAs' tiles through one descriptor
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(bg_smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char *a_tiles = base, *b_tiles = base + STAGES * BG_A_BYTES, *staging = b_tiles + STAGES * B_BYTES;
    BgCtrl* ctrl = reinterpret_cast<BgCtrl*>(staging + BG_WARPS * bg_staging<BN, OutT>());
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr bool SPLIT = BN == 128;
    const uint32_t cta = bg_cta_rank(), rank = SPLIT ? cta & 1u : cta, leader = SPLIT ? cta & ~1u : 0u;         // of the cluster, of its pair, and the pair's first
    const int split = (int)(cta >> 1), kb0 = SPLIT ? split * per : 0, n_kb = SPLIT ? min(per, k_blocks - kb0) : k_blocks, pair = blockIdx.y, pairs = gridDim.y;

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
                // the first stages' tiles of w before the kernel before this one has finished, where the caller says that it does not write them
                const int first = early ? min(STAGES, n_kb) : 0;
                const uint32_t full = bg_in_cta(&ctrl->full[0], leader);
                auto ask_w = [&](int s, int n0, int kb) {
                    if (rank == 0) bar_expect_tx(&ctrl->full[s], 2 * (BG_A_BYTES + B_BYTES));
                    bg_load_pair(b_tiles + s * B_BYTES, &map_w, (kb0 + kb) * QB, n0 + (int)rank * HALF, full + (uint32_t)s * 8u);
                };
                for (int kb = 0; kb < first; ++kb) ask_w(kb, (pair / m_tiles) * BN, kb);
                pdl_wait();
                int it = 0;
                for (int tile = pair; tile < num_tiles && !ctrl->abort; tile += pairs) {
                    const int n0 = (tile / m_tiles) * BN, m0 = (tile % m_tiles) * 2 * BG_M;
                    for (int kb = 0; kb < n_kb; ++kb, ++it) {
                        const int s = it % STAGES;
                        if (it >= STAGES && !bar_wait(&ctrl->empty[s], ((it / STAGES) - 1) & 1, &ctrl->abort)) break;
                        if (it >= first) ask_w(s, n0, kb);
                        bg_load_pair(a_tiles + s * BG_A_BYTES, &map_x, (kb0 + kb) * QB, m0 + (int)rank * BG_M, full + (uint32_t)s * 8u);
                    }
                }
            }
        } else if (warp == 1) {
            if (rank == 0) {
                // the whole warp walks the loop and waits, and leaves it together; one lane issues
                int it = 0;
                bool fine = true;
                for (int tile = pair; tile < num_tiles && fine; tile += pairs) {
                    for (int kb = 0; kb < n_kb; ++kb, ++it) {
                        const int s = it % STAGES, buf = it % BUFFERS;
                        if (!bar_wait_warp(&ctrl->full[s], (it / STAGES) & 1, &ctrl->abort)) { fine = false; break; }
                        const uint64_t adesc = smem_desc_sw128(a_tiles + s * BG_A_BYTES), bdesc = smem_desc_sw128(b_tiles + s * B_BYTES);
                        if (it >= BUFFERS && !bar_wait_warp(&ctrl->acc_empty[buf], ((it / BUFFERS) - 1) & 1, &ctrl->abort)) { fine = false; break; }
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        if (elect_one()) {
    #pragma unroll
                            for (int k = 0; k < QB / 32; ++k)          // 32 codes further along the swizzled row
                                umma_e4m3_pair(tmem_base + (uint32_t)(buf * BN), adesc + (uint64_t)(k * 32 >> 4), bdesc + (uint64_t)(k * 32 >> 4), IDESC, k != 0 ? 1u : 0u);
                            bg_commit_pair(&ctrl->empty[s], leader);
                            bg_commit_pair(&ctrl->acc_full[buf], leader);
                        }
                        __syncwarp();
                    }
                }
            }
        }
        if (SPLIT && splits > 1) {          // the epilogue's two meetings
            __syncwarp();
            cluster_sync_all();
            cluster_sync_all();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(BG_REGS_EPILOGUE));
        pdl_wait();
        // epilogue: warp w may touch TMEM lanes 32 * (w % 4) .. + 31; two warps share them, half of the columns each
        const int q = warp & 3, half = (warp - 4) / 4;
        const int n_blocks = (N + QB - 1) / QB;
        constexpr int COLS = bg_store_cols<OutT>(), STORE_BYTES = COLS * 32 * (int)sizeof(OutT), STAGED = bg_staging<BN, OutT>() / STORE_BYTES;
        unsigned char* mine = staging + (warp - 4) * bg_staging<BN, OutT>();
        const uint32_t released = bg_in_cta(&ctrl->acc_empty[0], leader);
        int it = 0;
        bool fine = true;
        for (int tile = pair; tile < num_tiles && fine; tile += pairs) {
            const int col0 = (tile / m_tiles) * BN + half * HALF, row0 = (tile % m_tiles) * 2 * BG_M + (int)rank * BG_M + q * 32, row = row0 + lane;
            // this warp's columns lie in one block of w's rows
            const float *pw = sw + (size_t)min(col0 / QB, n_blocks - 1) * k_blocks + kb0, *px = sx + min(row, M - 1) + (size_t)kb0 * M;
            unsigned long long acc[HALF / 2];
#pragma unroll
            for (int i = 0; i < HALF / 2; ++i) acc[i] = 0ull;
            // the scales of two blocks ahead are on their way: a block takes less time than a load from memory
            float a[2], b[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int kb = min(i, n_kb - 1);
                a[i] = px[(size_t)kb * M];
                b[i] = pw[kb];
            }
#pragma unroll 2
            for (int kb = 0; kb < n_kb; ++kb, ++it) {
                const int buf = it % BUFFERS;
                const unsigned long long s2 = twice(a[kb & 1] * b[kb & 1]);
                if (kb + 2 < n_kb) {
                    a[kb & 1] = px[(size_t)(kb + 2) * M];
                    b[kb & 1] = pw[kb + 2];
                }
                if (!bar_wait_warp(&ctrl->acc_full[buf], (it / BUFFERS) & 1, &ctrl->abort)) { fine = false; break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t from = tmem_base + (uint32_t)(buf * BN + half * HALF) + ((uint32_t)(q * 32) << 16);
#pragma unroll
                for (int c = 0; c < HALF / 32; ++c) {
                    uint32_t r[32];
                    tmem_ld32_pinned(from + (uint32_t)(c * 32), r);
                    if (c + 1 == HALF / 32) {
                        // this warp has read its lanes of the accumulator: CTA 0's product warp may write it again
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) bg_arrive_cluster(released + (uint32_t)buf * 8u);
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) fma2(acc[c * 16 + i], r[2 * i], r[2 * i + 1], s2);
                }
            }
            if (SPLIT && splits > 1) {
                // every pair is done with its products and copies: the first one's stages hold the others' sums, [split][4 columns][row][column of 4]
                cluster_sync_all();
                float4* sums = reinterpret_cast<float4*>(base) + ((half * (HALF / 4)) * BG_M + q * 32 + lane);
                if (split > 0) {
                    const uint32_t to = bg_in_cta(sums + (size_t)(split - 1) * (BN / 4) * BG_M, rank);
#pragma unroll
                    for (int c = 0; c < HALF / 4; ++c) {
                        const float2 v = two_of(acc[2 * c]), w = two_of(acc[2 * c + 1]);
                        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to + (uint32_t)(c * BG_M * 16)), "f"(v.x), "f"(v.y), "f"(w.x), "f"(w.y) : "memory");
                    }
                }
                cluster_sync_all();
                if (split > 0) break;
                for (int o = 1; o < splits; ++o) {
#pragma unroll
                    for (int c = 0; c < HALF / 4; ++c) {
                        const float4 v = sums[((size_t)(o - 1) * (BN / 4) + c) * BG_M];
                        add2(acc[2 * c], v.x, v.y);
                        add2(acc[2 * c + 1], v.z, v.w);
                    }
                }
            }
            if (!fine) break;
#pragma unroll
            for (int c = 0; c < HALF / COLS; ++c) {
                if (c % STAGED == 0) {
                    // what the last stores read has to be read before it is written over
                    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                    __syncwarp();
                }
                unsigned char* to = mine + (c % STAGED) * STORE_BYTES;
                stage_sums<COLS, OutT>(acc + c * (COLS / 2), reinterpret_cast<uint4*>(to));
                if (bulk_stores) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0 && row0 < M && col0 + c * COLS < N) {
                        tma_store_2d(&map_y, to, col0 + c * COLS, row0);
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                } else {
                    __syncwarp();
                    store_staged<COLS, OutT>(reinterpret_cast<const uint4*>(to), y, row0, col0 + c * COLS, M, N);
                    __syncwarp();
                }
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
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

// The result [M, N] as a tensor map with boxes of 32 rows x cols columns, in the layout of stage_sums.
template <typename OutT> bool make_result_map(CUtensorMap* map, void* y, int M, int N, int cols) {
    EncodeTiledFn fn = encode_fn();
    if (fn == nullptr) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)N, (cuuint64_t)M};
    const cuuint64_t strides[1] = {(cuuint64_t)N * sizeof(OutT)};
    const cuuint32_t box[2] = {(cuuint32_t)cols, 32u};
    const cuuint32_t estr[2] = {1, 1};
    return fn(map, sizeof(OutT) == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, y, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BN, typename OutT>
int launch_blocks_gemm(const void* x, long long ldx, const float* sx, const void* w, long long ldw, const float* sw, void* y, int M, int N, int K, int splits,
                       int early, int sms, cudaStream_t stream) {
    static std::atomic<unsigned long long> allowed{0};
    const cudaError_t e = rlis_allow_smem(blocks_gemm_kernel<BN, OutT>, (int)bg_smem<BN, OutT>(), allowed);
    if (e != cudaSuccess) return (int)e;
    CUtensorMap map_x, map_w, map_y;
    if (!make_code_map(&map_x, x, M, K, BG_M, ldx) || !make_code_map(&map_w, w, N, K, BN / 2, ldw)) return RLIS_ERR_UNSUPPORTED;
    // rows of the result that start at multiples of 16 bytes leave by bulk tensor copies
    const bool bulk = ((long long)N * (int)sizeof(OutT)) % 16 == 0 && (reinterpret_cast<uintptr_t>(y) & 15) == 0;
    map_y = map_x;
    if (bulk && !make_result_map<OutT>(&map_y, y, M, N, bg_store_cols<OutT>())) return RLIS_ERR_UNSUPPORTED;
    const int m_tiles = (M + 2 * BG_M - 1) / (2 * BG_M), num_tiles = m_tiles * ((N + BN - 1) / BN), k_blocks = (K + QB - 1) / QB;
    const int per = (k_blocks + splits - 1) / splits;
    splits = (k_blocks + per - 1) / per;                // none without a block
    const int pairs = splits > 1 || num_tiles < sms / 2 ? num_tiles : sms / 2;
    rlis_launch_cluster(blocks_gemm_kernel<BN, OutT>, dim3(2u * splits, (unsigned)pairs), dim3(BG_THREADS), bg_smem<BN, OutT>(), stream, dim3(2u * splits, 1, 1), map_x,
                        map_w, map_y, sx, sw, (OutT*)y, M, N, k_blocks, per, m_tiles, num_tiles, splits, bulk ? 1 : 0, early);
    return RLIS_LAUNCH_CHECK();
}
}  // namespace

#include "blocks_few.cuh"

// 0 if no bounded wait of these products ever ran out on the current device.
extern "C" int rlis_blocks_gemm_error(void) { return tc::read_error_word(); }
extern "C" int* rlis_blocks_gemm_error_addr(void) { return tc::error_word_addr(); }

namespace {
int sms_of_device() {
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms;
}
constexpr int FEW_ROWS = 128;           // rows up to which a product is a stream of w
bool codes_fit(const void* p, long long ld, int K) { return ld >= K && ld % 16 == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
}  // namespace

// x [M, K] (rows ldx bytes apart), sx [ceil(K / 128), M]; w [N, K] (rows ldw bytes apart), sw [ceil(N / 128), ceil(K / 128)]; y [M, N].  Codes on 16-byte
// boundaries, their rows multiples of 16 bytes apart.  early: no kernel still in flight writes w, so that its first tiles may be read before the kernel before
// this one has finished.
extern "C" int rlis_blocks_gemm(const void* x, long long ldx, const float* sx, const void* w, long long ldw, const float* sw, void* y, int M, int N, int K, int out_dtype,
                                int early, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0 || (out_dtype != RLIS_F32 && out_dtype != RLIS_BF16) || !codes_fit(x, ldx, K) || !codes_fit(w, ldw, K)) return RLIS_ERR_UNSUPPORTED;
    const int sms = sms_of_device();
    const bool f32 = out_dtype == RLIS_F32;
    if (M <= FEW_ROWS) {
#define RLIS_BF(NT) (f32 ? launch_blocks_few<NT, float>(x, ldx, sx, w, ldw, sw, y, M, N, K, early, sms, stream) \
                         : launch_blocks_few<NT, bf16>(x, ldx, sx, w, ldw, sw, y, M, N, K, early, sms, stream))
        return M <= 16 ? RLIS_BF(16) : M <= 32 ? RLIS_BF(32) : M <= 64 ? RLIS_BF(64) : RLIS_BF(128);
#undef RLIS_BF
    }
    // The width of a tile: a round of 128 columns over the pairs of SMs takes 0.8 of one of 256 (as many steps along k, each waiting for the sums before it), so the
    // narrow ones pay only where they need no more rounds (us in 128 / 256 columns: 512 x 4,096 of K 4096, one round either way, 14.9 / 17.8; 509 x 6,100 of K 4000,
    // two rounds or one, 29.5 / 21.4; 1,024 x 14,336 of K 4096 73.4 / 61.1; 192 columns were slower than one of the two at all of 13 sizes).
    const long long m_tiles = (M + 2 * BG_M - 1) / (2 * BG_M), pairs = sms / 2;
    auto rounds = [&](int bn) { return (m_tiles * ((N + bn - 1) / bn) + pairs - 1) / pairs; };
    const bool wide = 4 * rounds(128) >= 5 * rounds(256);
    // The pairs that a round of narrow tiles leaves idle take shares of k, where that shortens it by 12 blocks or more: a block is 0.3 us, the meeting of the sums 3
    // (us in 1 / 2 / 3 shares: 129 x 4,096 of K 14336 37.2 / 25.3 / more than the pairs; 256 x 2,048 of K 8192 23.2 / 17.2 / 15.4; 129 x 1,024 of K 4096 13.5 / 11.5 /
    // 10.9; 300 x 2,048 of K 2048, where 2 shares save 8 blocks, 9.2 / 9.8).
    const int k_blocks = (K + QB - 1) / QB;
    int splits = wide ? 1 : (int)std::min<long long>(BG_MAX_SPLITS, std::max<long long>(1, pairs / (m_tiles * ((N + 127) / 128))));
    if (k_blocks - (k_blocks + splits - 1) / splits < 12) splits = 1;
#define RLIS_BG(BN) (f32 ? launch_blocks_gemm<BN, float>(x, ldx, sx, w, ldw, sw, y, M, N, K, splits, early, sms, stream) \
                         : launch_blocks_gemm<BN, bf16>(x, ldx, sx, w, ldw, sw, y, M, N, K, splits, early, sms, stream))
    return wide ? RLIS_BG(256) : RLIS_BG(128);
#undef RLIS_BG
}

extern "C" int rlis_quantize_rows(const void* x, long long ldx, void* codes, long long ldc, float* scales, int n_tokens, int K, int dtype, cudaStream_t stream);

// The bytes of scratch that rlis_blocks_gemm_rows wants on the current device: 0 where the product puts the rows into blocks itself.
extern "C" long long rlis_blocks_gemm_scratch(int M, int N, int K) {
    if (M <= 0 || N <= 0 || K <= 0 || plain_rows_fit(M, N, K, sms_of_device())) return 0;
    return M * ((K + 15LL) / 16 * 16 + 4LL * ((K + QB - 1) / QB));
}

// The same for plain rows x [M, K] of `dtype` (ldx elements apart), which the product puts into blocks itself or rlis_quantize_rows before it.  scratch: 16-byte aligned,
// M * ceil(K / 16) * 16 bytes of codes and behind them M * ceil(K / 128) floats.  early: as above for one kernel.  (Of two the first lets the second start once all
// kernels before itself have finished; none but itself is in flight then, and it does not write w: w's first tiles are always read early.)
extern "C" int rlis_blocks_gemm_rows(const void* x, long long ldx, int dtype, void* scratch, const void* w, long long ldw, const float* sw, void* y, int M, int N, int K,
                                     int out_dtype, int early, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0) return RLIS_ERR_UNSUPPORTED;
    const int sms = sms_of_device();
    if (plain_rows_fit(M, N, K, sms)) {
        if ((dtype != RLIS_F32 && dtype != RLIS_BF16) || (out_dtype != RLIS_F32 && out_dtype != RLIS_BF16) || !codes_fit(w, ldw, K)) return RLIS_ERR_UNSUPPORTED;
#define RLIS_BP(T) (out_dtype == RLIS_F32 ? launch_blocks_few_plain<T, float>(x, ldx, w, ldw, sw, y, M, N, K, early, sms, stream) \
                                          : launch_blocks_few_plain<T, bf16>(x, ldx, w, ldw, sw, y, M, N, K, early, sms, stream))
        return dtype == RLIS_F32 ? RLIS_BP(float) : RLIS_BP(bf16);
#undef RLIS_BP
    }
    if (scratch == nullptr) return RLIS_ERR_UNSUPPORTED;
    const long long ldc = (K + 15LL) / 16 * 16;
    float* sx = reinterpret_cast<float*>(static_cast<unsigned char*>(scratch) + M * ldc);
    const int e = rlis_quantize_rows(x, ldx, scratch, ldc, sx, M, K, dtype, stream);
    return e != 0 ? e : rlis_blocks_gemm(scratch, ldc, sx, w, ldw, sw, y, M, N, K, out_dtype, 1, stream);
}
