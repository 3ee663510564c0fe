// A whole mixture of experts for up to 16 tokens in two kernels (moe.cu says what each part of it computes):
//
//   up:   z = W_r x, the choice of `top` outputs a token and their weights; h[t, e, :] = weight[t, e] glu(W_gate_e x_t, W_up_e x_t) for the chosen pairs, and
//         h[t, s, :] = gate[t] glu(..) of the shared expert
//   down: out[t, :] = sum over e of W_down_e h[t, e, :] (+ W_down_s h[t, s, :]) + sum of the weights of t's identity experts * x_t
//
// With so few tokens the layer is a stream of the chosen experts' weights from memory (8 tokens, 4 of 32 experts of 2,048 x 1,024 and a shared one: 290 MB, 44 us
// at the rate of a copy; the two kernels take 63).  So every weight is read once, by 16-byte loads of 16 rows side by side straight into the registers of mma.sync
// m16n8k16, no shared memory between: a sum over k may take k in any order, so a thread's 16 bytes of a row, eight neighbouring k, serve as its k slots of two
// instructions, and the tokens' rows are read in the same order.  A warp takes 128 k of 16 rows at a time (a chunk, a block's edge; for weights in e4m3 blocks a
// chunk's sums are scaled before they join the others) and has the next chunks, of the next rows if need be, on their way while it works on one.  The warps of a
// team take different k of the same rows and add their sums in shared memory in the order of the warps, so results do not depend on timing.  In flight the loads
// take room in the first-level cache, which is what shared memory leaves: chunks by asynchronous copies through 180 KB of shared memory took 99 us for 65, and the
// down kernel with 227 KB instead of 163 353 for 179.
//
// Routing sits in the up kernel: the CTAs of a cluster share the router's rows, hand each other the logits (distributed shared memory), and each chooses
// for all tokens itself: no launch of its own, no grid-wide barrier, no workspace but h, the plan, which the first CTA leaves for the down kernel, and a copy of
// the tokens' rows for each cluster, which the caches hold.  The router's float32 rows go through the same instructions as three bfloat16 numbers each, whose sum
// they are to 2^-24 (a token's logits are sums of exact products in float32, as a chain of FMAs would give them; as FMAs, 128 rows against 16 tokens took 20 us).
//
// The weights of the choice are multiplied into h in float32; the down product is then one long sum over the chosen experts' k, with the step's tokens as columns
// whoever chose them.  Its CTAs bring the pieces of h that their chunks meet into shared memory first (read from the second-level cache chunk by chunk they took
// more of the load units than the weights: 16 tokens, 83 of 128 experts of 768 in blocks 135 us, 111 so, each with one number of float16 for h).
// Nothing but the result is rounded to the activations' type: beside bfloat16 weights h is two bfloat16 numbers (their sum is h to 2^-17).  Codes become float16 by one instruction a pair (as bfloat16, which has none,
// a word of four took 10 cycles of a scheduler instead of 5, and the products waited for it), so the tokens' rows and h's meet them as float16 of eleven bits, each
// row (of h each piece of 128) times the power of two that brings its largest value to 2^14 .. 2^15: x is that exactly down to 2^-31 of the largest, h is two such
// numbers, whose sum is h to 2^-22, or 2^-39 of the piece's largest.  (One of them is h to 2^-11 and takes 112 us for 121 in that layer, 41.3 for 43.6 with 8 tokens; but its
// results are up to 9e-4 away from those of float32, and two numbers' 5e-5 as sums in another order are.)
//
// What bounds it: memory in the two loops (8 tokens in bfloat16: 6.8 TB/s), and what comes before and between them, when memory is idle: 8 us from the launch
// to the first expert's weights (the router's rows, the meeting of the cluster, the choice), 4 from the first CTA's last item to the down kernel's plan, 4 to its first
// product, 2 for the last sums.
#include "common.cuh"
#include "mma_utils.cuh"
#include <cuda_fp16.h>
#include <math.h>

namespace {
constexpr int LT = 16;                  // tokens
constexpr int L_WARPS = 16, L_THREADS = 32 * L_WARPS;
constexpr int L_CLUSTER = 8;            // CTAs that share the router's rows
constexpr int L_MAX_OUT = 512;          // router outputs
constexpr int L_MAX_PAIRS = 256;        // tokens * top
constexpr int LK = 128;                 // k of a chunk
constexpr int MOST_K = 16384;           // of a matrix of the layer (items' numbers stay within what a product divides)

// An expert that some token chose: the tokens as bits, as a list (four bits each), and which of a token's choices it is (four bits a token).
constexpr unsigned SECOND = 0x8000u;
struct ActiveExpert {
    int expert;
    unsigned tokens;
    unsigned long long list, choice;
};
// What the up kernel leaves for the down kernel: the active experts, ascending.
struct LayerPlan {
    int n_active, unused;
    float identity[LT];                 // a token's weights of identity experts, summed
    ActiveExpert of[L_MAX_PAIRS];
};

// One matrix of the layer (or a stack): `ld` elements (bfloat16) or bytes (codes) between rows; codes have scales [matrix][row / 128][k / 128].
struct LayerMatrix {
    const unsigned char* w;
    const float* scales;
    long long row_bytes, stack_bytes;
    int row_blocks, k_blocks;
};

struct LayerArgs {
    const bf16* x;
    long long ldx;
    int n_tokens, width;
    const float *router, *correction, *router_bias;
    int n_out, n_real, top, scoring, n_groups, keep_groups, normalize, shared_gate;
    float route_scale;
    int inner, inner_shared, interleave, interleave_shared;        // inner_shared 0: no shared expert
    LayerMatrix up, down, shared_up, shared_down;
    float slope, limit, shift;
    LayerPlan* plan;
    bf16 *h_hi, *h_lo;                  // [tokens * top + tokens, h_row]: the pairs', the shared expert's; or, beside codes, float32:
    float* h;
    bf16* x_copy;                       // [cluster of the up kernel][tokens][x_row] (float16 beside codes)
    int x_row, h_row;
    unsigned per_expert_magic, own_chunks_magic;        // see quotient()
    bf16* out;
};

// n / d with d's magic number ceil(2^32 / d) (0 for d 1), exact for n below 2^32 / d.
__device__ __forceinline__ int quotient(int n, unsigned magic) { return magic != 0u ? (int)__umulhi((unsigned)n, magic) : n; }

__device__ __forceinline__ uint4 stream16(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// Four codes as float16, in their order.
__device__ __forceinline__ void widen_codes(uint32_t w, uint32_t& first, uint32_t& last) {
    asm("{\n"
        ".reg .b16 lo, hi;\n"
        "mov.b32 {lo, hi}, %2;\n"
        "cvt.rn.f16x2.e4m3x2 %0, lo;\n"
        "cvt.rn.f16x2.e4m3x2 %1, hi;\n"
        "}\n"
        : "=r"(first), "=r"(last) : "r"(w));
}
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool CODES> __device__ __forceinline__ void mma_step(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (CODES) mma_f16_16816(d, a, b0, b1);
    else mma_bf16_16816(d, a, b0, b1);
}

// 128 k of rows g and g + 8 of a warp's 16 (g = lane / 4): lane % 4 holds every fourth 16 bytes.
template <bool CODES> struct Chunk {
    static constexpr int STEPS = CODES ? 2 : 4, PARTS = CODES ? 4 : 2;         // instructions a step
    uint4 a[STEPS][2];
    float scale[2];             // codes: of row g, of row g + 8
    __device__ __forceinline__ void operand(int s, int j, uint32_t (&to)[4]) const {
        const uint32_t r0[4] = {a[s][0].x, a[s][0].y, a[s][0].z, a[s][0].w}, r1[4] = {a[s][1].x, a[s][1].y, a[s][1].z, a[s][1].w};
        if constexpr (CODES) {
            widen_codes(r0[j], to[0], to[2]);
            widen_codes(r1[j], to[1], to[3]);
        } else {
            to[0] = r0[2 * j], to[1] = r1[2 * j], to[2] = r0[2 * j + 1], to[3] = r1[2 * j + 1];
        }
    }
};
__device__ const uint4 NOTHING = {0u, 0u, 0u, 0u};
// `row0`, `row1`: this lane's rows of K; the chunk is k0 .. k0 + 127.  The columns' rows are padded with zeros, so that no chunk needs code of its own: of what lies past
// the row's end, codes are its last 16 bytes again (a NaN among them has made the sum one already), and bfloat16 are zeros (an infinity would make a NaN of it).
template <bool CODES>
__device__ __forceinline__ void load_chunk(Chunk<CODES>& c, const unsigned char* row0, const unsigned char* row1, int k0, int K, int lane) {
    constexpr int PER = CODES ? 16 : 8;
#pragma unroll
    for (int s = 0; s < Chunk<CODES>::STEPS; ++s) {
        const int k = k0 + (s * 4 + (lane & 3)) * PER;
        if (CODES) {
            const int at = min(k, K - PER);
            c.a[s][0] = stream16(row0 + at);
            c.a[s][1] = stream16(row1 + at);
        } else {
            c.a[s][0] = stream16(k < K ? row0 + 2 * k : reinterpret_cast<const unsigned char*>(&NOTHING));
            c.a[s][1] = stream16(k < K ? row1 + 2 * k : reinterpret_cast<const unsigned char*>(&NOTHING));
        }
    }
}

// The powers of two that bring a row whose largest float32 exponent is e (biased) to 2^14 .. 2^15 and back; rows below 2^-112 stay below that.
constexpr int LEAST_EXPONENT = 15;
__device__ __forceinline__ float scaling_of(int e) { return __uint_as_float((unsigned)(268 - e) << 23); }
__device__ __forceinline__ float unscaling_of(int e) { return __uint_as_float((unsigned)(e - 14) << 23); }
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// Two numbers as float16 and what these leave of them.
__device__ __forceinline__ void split_half(float a, float b, uint32_t& first, uint32_t& rest) {
    const __half2 v = __floats2half2_rn(a, b);
    const float2 f = __half22float2(v);
    first = *reinterpret_cast<const uint32_t*>(&v);
    rest = pack_half(a - f.x, b - f.y);
}

// This lane's part of a column's row over a chunk: the vectors of bfloat16 that its A vectors meet.
template <bool CODES> struct Column {
    static constexpr int VECS = CODES ? 2 : 1;
    uint4 b[Chunk<CODES>::STEPS][VECS];
};
// `row`: the column's row from this lane's first k of the chunk on.
template <bool CODES> __device__ __forceinline__ void load_column(Column<CODES>& c, const bf16* row) {
#pragma unroll
    for (int s = 0; s < Chunk<CODES>::STEPS; ++s)
#pragma unroll
        for (int v = 0; v < Column<CODES>::VECS; ++v) c.b[s][v] = *reinterpret_cast<const uint4*>(row + s * (CODES ? 64 : 32) + v * 8);
}
// acc += chunk * column.  Neighbouring instructions add to different sums: one waits some 35 cycles for the one before it on the same.
template <bool CODES> __device__ __forceinline__ void multiply(const Chunk<CODES>& c, const Column<CODES>& col, float (&acc)[4]) {
    float part[2][4] = {};
#pragma unroll
    for (int s = 0; s < Chunk<CODES>::STEPS; ++s) {
#pragma unroll
        for (int j = 0; j < Chunk<CODES>::PARTS; ++j) {
            uint32_t a[4];
            c.operand(s, j, a);
            const uint4 b = col.b[s][CODES ? j / 2 : 0];
            mma_step<CODES>(part[j & 1], a, j & 1 ? b.z : b.x, j & 1 ? b.w : b.y);
        }
    }
    const float s0 = CODES ? c.scale[0] : 1.f, s1 = CODES ? c.scale[1] : 1.f;
    acc[0] = fmaf(part[0][0] + part[1][0], s0, acc[0]);
    acc[1] = fmaf(part[0][1] + part[1][1], s0, acc[1]);
    acc[2] = fmaf(part[0][2] + part[1][2], s1, acc[2]);
    acc[3] = fmaf(part[0][3] + part[1][3], s1, acc[3]);
}

// ---- the choice ------------------------------------------------------------------------------------------------------------------------

// Bits that order floats as unsigned numbers; 0: a NaN, which is never chosen.  (-0 counts as 0.)
__device__ __forceinline__ unsigned order_of(float v) {
    if (v != v) return 0u;
    const unsigned b = __float_as_uint(v + 0.f);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logistic(float z) { return 1.0f / (1.0f + expf(-z)); }

// One warp chooses for one token: z [n_out] logits in, scores out; `key` [n_out + n_groups] is scratch.  Lane k ends with choice k and its weight.
__device__ __forceinline__ void choose(const LayerArgs& p, const float* correction, const float* bias, float* z, unsigned* key, int lane, int& chosen, float& weight) {
    const int n = p.n_out;
    float mx = -INFINITY;
    if (p.scoring == 2) {
#pragma unroll 1
        for (int e = lane; e < n; e += 32) mx = fmaxf(mx, z[e] + bias[e]);
        mx = warp_max(mx);
    }
    float sum = 0.f;
#pragma unroll 1
    for (int e = lane; e < n; e += 32) {
        float v = z[e] + bias[e];
        if (p.scoring != 1) v = expf(p.scoring == 2 ? v - mx : -v);
        if (p.scoring == 0) v = 1.0f / (1.0f + v);
        sum += v;
        z[e] = v;
    }
    if (p.scoring == 2) sum = warp_sum(sum);
#pragma unroll 1
    for (int e = lane; e < n; e += 32) {
        const float v = p.scoring == 2 ? z[e] / sum : z[e];
        z[e] = v;
        key[e] = order_of(v + correction[e]);
    }
    __syncwarp();
    if (p.n_groups > 1) {
        // a group's rank is its best choice score; a group is kept when fewer than keep_groups rank before it (ties: the lower one first)
        const int per = n / p.n_groups;
        unsigned* best = key + n;
        for (int g = lane; g < p.n_groups; g += 32) {
            unsigned m = 0u;
            for (int e = g * per; e < (g + 1) * per; ++e) m = max(m, key[e]);
            best[g] = m;
        }
        __syncwarp();
        for (int g = lane; g < p.n_groups; g += 32) {
            int before = 0;
            for (int o = 0; o < p.n_groups; ++o) before += best[o] > best[g] || (best[o] == best[g] && o < g);
            if (before >= p.keep_groups)
                for (int e = g * per; e < (g + 1) * per; ++e) key[e] = 0u;
        }
        __syncwarp();
    }
    chosen = 0;
    weight = 0.f;
    unsigned taken = 0u;            // this lane's outputs (lane + 32 i: bit i) that are chosen
#pragma unroll 1
    for (int k = 0; k < p.top; ++k) {
        unsigned best = 0u;
        int at = 0;
#pragma unroll 4
        for (int i = 0; i * 32 < n; ++i) {
            const int e = lane + 32 * i;
            const unsigned v = e < n ? key[e] : 0u;
            if (v > best) {
                best = v;
                at = e;
            }
        }
        const unsigned m = __reduce_max_sync(0xffffffffu, best);
        // (where nothing is left that compares, the first output that is not chosen yet)
        const int open = 32 * (__ffs((int)~taken) - 1) + lane;
        const unsigned e = __reduce_min_sync(0xffffffffu, m != 0u ? best == m ? (unsigned)at : 0xffffffffu : open < n ? (unsigned)open : 0xffffffffu);
        if (lane == (int)(e & 31u)) {
            taken |= 1u << (e >> 5);
            key[e] = 0u;
        }
        if (lane == k) {
            chosen = (int)e;
            weight = z[e];
        }
    }
    const bool mine = lane < p.top;
    if (p.scoring == 1) {               // the softmax over the chosen logits
        const float most = warp_max(mine ? weight : -INFINITY), v = mine ? expf(weight - most) : 0.f;
        weight = v / warp_sum(v) * p.route_scale;
    } else {
        weight = p.normalize ? weight / (warp_sum(mine ? weight : 0.f) + 1e-20f) * p.route_scale : weight * p.route_scale;
    }
}

// A float into the shared memory of the cluster's CTA `rank` (at the offset of `local`); a cluster barrier orders it before the reads.
__device__ __forceinline__ void st_cluster_f32(float* local, float v, uint32_t rank) {
    uint32_t raddr;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(raddr) : "r"(smem_u32(local)), "r"(rank));
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(raddr), "f"(v) : "memory");
}

// ---- up --------------------------------------------------------------------------------------------------------------------------------

constexpr int MOST_TEAM = 8;                                // warps that share an item's k: 4 or 8 (see launch_layer)
static_assert(L_WARPS <= 16, "a barrier for each team and set");

template <int GROUPS, int TEAM> struct UpShared {
    union {                                     // the warps' sums of 16 rows, sets in turn
        float router[2][L_WARPS][16][8 * GROUPS + 1];
        float reduce[TEAM][L_WARPS][16][8 + 1];
    };
    LayerPlan plan;
    float gate[LT];
    int exponent[LT];                           // beside codes: the largest exponent of a token's row
    unsigned top[L_WARPS];
    unsigned long long choice[L_MAX_OUT];       // which of a token's choices an expert is, four bits a token
    unsigned tokens[L_MAX_OUT];                 // the tokens that chose an expert
    float correction[L_MAX_OUT], bias[L_MAX_OUT];       // of the outputs (zeros where there are none): on their way with the router's rows
    unsigned short work[2 * L_MAX_PAIRS];       // active experts, with SECOND set for those after the first eight of an expert's tokens
};

// This CTA's rows of the router against all tokens, into every CTA's z [LT][z_row].  Sixteen rows at a time; the warps share k: a warp takes 128 k of the
// sixteen rows as three bfloat16 each.
template <int GROUPS, int TEAM>
__device__ __forceinline__ void router_logits(const LayerArgs& p, UpShared<GROUPS, TEAM>& sh, float* z, int z_row, int rank, int cluster) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2;
    const int rows = p.n_out + p.shared_gate, per = (rows + cluster - 1) / cluster, first = rank * per, mine = max(0, min(per, rows - first));
    const int tiles = (per + 15) / 16, n_chunks = (p.width + LK - 1) / LK;
    bool met = false;
    for (int tile = 0; tile < tiles; ++tile) {
        float acc[GROUPS][4] = {};
        const int r0 = tile * 16 + g, r1 = r0 + 8;
        const float *w0 = p.router + (long long)(first + min(r0, mine - 1)) * p.width, *w1 = p.router + (long long)(first + min(r1, mine - 1)) * p.width;
        for (int chunk = warp; chunk < n_chunks && tile * 16 < mine; chunk += L_WARPS) {
            const int k0 = chunk * LK + (lane & 3) * 8;
            float4 a[4][2][2];
            uint4 x[4][GROUPS];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int k = k0 + s * 32;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    a[s][0][h] = k < p.width ? *reinterpret_cast<const float4*>(w0 + k + 4 * h) : make_float4(0, 0, 0, 0);
                    a[s][1][h] = k < p.width ? *reinterpret_cast<const float4*>(w1 + k + 4 * h) : make_float4(0, 0, 0, 0);
                }
#pragma unroll
                for (int n = 0; n < GROUPS; ++n)
                    x[s][n] = k < p.width && n * 8 + g < p.n_tokens ? *reinterpret_cast<const uint4*>(p.x + (n * 8 + g) * p.ldx + k) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                float v[2][8];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    v[r][0] = a[s][r][0].x, v[r][1] = a[s][r][0].y, v[r][2] = a[s][r][0].z, v[r][3] = a[s][r][0].w;
                    v[r][4] = a[s][r][1].x, v[r][5] = a[s][r][1].y, v[r][6] = a[s][r][1].z, v[r][7] = a[s][r][1].w;
                }
#pragma unroll 1
                for (int part = 0; part < 3; ++part) {
                    uint32_t w[2][4];
#pragma unroll
                    for (int r = 0; r < 2; ++r)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            w[r][i] = pack_bf16(v[r][2 * i], v[r][2 * i + 1]);
                            v[r][2 * i] -= __uint_as_float(w[r][i] << 16);
                            v[r][2 * i + 1] -= __uint_as_float(w[r][i] & 0xffff0000u);
                        }
                    const uint32_t a0[4] = {w[0][0], w[1][0], w[0][1], w[1][1]}, a1[4] = {w[0][2], w[1][2], w[0][3], w[1][3]};
#pragma unroll
                    for (int n = 0; n < GROUPS; ++n) {
                        mma_bf16_16816(acc[n], a0, x[s][n].x, x[s][n].y);
                        mma_bf16_16816(acc[n], a1, x[s][n].z, x[s][n].w);
                    }
                }
            }
        }
        auto& sums = sh.router[tile & 1][warp];
        const int col = (lane & 3) * 2;
#pragma unroll
        for (int n = 0; n < GROUPS; ++n) {
            sums[g][n * 8 + col] = acc[n][0];
            sums[g][n * 8 + col + 1] = acc[n][1];
            sums[g + 8][n * 8 + col] = acc[n][2];
            sums[g + 8][n * 8 + col + 1] = acc[n][3];
        }
        __syncthreads();
        if (!met) {                     // every CTA of the cluster has begun before its shared memory is written from another
            asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
            met = true;
        }
        if (threadIdx.x < 16 * LT) {
            const int r = threadIdx.x / LT, t = threadIdx.x % LT;
            if (tile * 16 + r < mine && t < p.n_tokens) {
                float v = 0.f;
#pragma unroll
                for (int i = 0; i < L_WARPS; ++i) v += sh.router[tile & 1][i][r][t];
                for (int c = 0; c < cluster; ++c) st_cluster_f32(z + t * z_row + first + tile * 16 + r, v, (uint32_t)c);
            }
        }
    }
}

// The cluster's copy of the tokens' rows, padded with zeros to x_row; beside codes as scaled float16, and their exponents in every CTA.  Eight warps a token.
template <bool CODES, int GROUPS, int TEAM>
__device__ __forceinline__ void copy_rows(const LayerArgs& p, UpShared<GROUPS, TEAM>& sh, bf16* to, int rank, const uint4 head) {
    static_assert(L_CLUSTER * 2 >= LT && L_WARPS == 16, "two tokens a CTA at the most");
    const int warp = threadIdx.x >> 5, t = rank + L_CLUSTER * (warp >> 3), i0 = threadIdx.x & 255;
    const bf16* x = p.x + (long long)min(t, p.n_tokens - 1) * p.ldx;
    int e = 0;
    if (CODES) {
        unsigned m = 0u;
        for (int k = i0 * 8; k < p.width; k += 2048) {
            const uint4 v = k == i0 * 8 ? head : *reinterpret_cast<const uint4*>(x + k);
            m = __vmaxu2(__vmaxu2(m, __vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu)), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
        }
        m = __reduce_max_sync(0xffffffffu, max(m & 0xffffu, m >> 16));
        if ((threadIdx.x & 31) == 0) sh.top[warp] = m;
        __syncthreads();
        for (int w = 0; w < 8; ++w) m = max(m, sh.top[(warp & 8) + w]);
        e = max((int)(m >> 7), LEAST_EXPONENT);
    }
    if (t >= p.n_tokens) return;
    const float scaling = scaling_of(e);
#pragma unroll 1
    for (int k = i0 * 8; k < p.x_row; k += 2048) {
        uint4 v = k == i0 * 8 ? head : k < p.width ? *reinterpret_cast<const uint4*>(x + k) : make_uint4(0, 0, 0, 0);
        if (CODES) {
            auto two = [&](uint32_t w) { return pack_half(__uint_as_float(w << 16) * scaling, __uint_as_float(w & 0xffff0000u) * scaling); };
            v = make_uint4(two(v.x), two(v.y), two(v.z), two(v.w));
        }
        *reinterpret_cast<uint4*>(to + (long long)t * p.x_row + k) = v;
    }
    if (CODES && i0 < L_CLUSTER) st_cluster_f32(reinterpret_cast<float*>(&sh.exponent[t]), __int_as_float(e), (uint32_t)i0);
}

template <bool CODES, int GROUPS /* of eight tokens */, int TEAM>
__global__ __launch_bounds__(L_THREADS, 1) void moe_layer_up_kernel(const LayerArgs p) {
    extern __shared__ __align__(16) unsigned char up_smem[];
    constexpr int TEAMS = L_WARPS / TEAM;
    using Shared = UpShared<GROUPS, TEAM>;
    Shared& sh = *reinterpret_cast<Shared*>(up_smem);
    float* z = reinterpret_cast<float*>(up_smem + sizeof(Shared));                     // [LT][z_row]: logits, later the weights of what was chosen
    const int z_row = p.n_out + 1;
    unsigned* keys = reinterpret_cast<unsigned*>(z + LT * z_row);                        // [LT][n_out + n_groups]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2;
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    for (int e = threadIdx.x; e < p.n_out; e += L_THREADS) {
        sh.tokens[e] = 0u;
        sh.choice[e] = 0ull;
    }
    pdl_wait();
    for (int e = threadIdx.x; e < p.n_out; e += L_THREADS) {
        sh.correction[e] = p.correction != nullptr ? p.correction[e] : 0.f;
        sh.bias[e] = p.router_bias != nullptr ? p.router_bias[e] : 0.f;
    }
    // (the first of this thread's vectors of the tokens' rows that copy_rows copies: on its way meanwhile)
    const int copied = min((int)(blockIdx.x % L_CLUSTER) + L_CLUSTER * (warp >> 3), p.n_tokens - 1), head_k = (threadIdx.x & 255) * 8;
    const uint4 head = head_k < p.width ? *reinterpret_cast<const uint4*>(p.x + copied * p.ldx + head_k) : make_uint4(0, 0, 0, 0);
    router_logits(p, sh, z, z_row, blockIdx.x % L_CLUSTER, L_CLUSTER);
    bf16* x_copy = p.x_copy + (long long)(blockIdx.x / L_CLUSTER) * p.n_tokens * p.x_row;
    copy_rows<CODES>(p, sh, x_copy, blockIdx.x % L_CLUSTER, head);
    cluster_sync_all();

    if (warp < p.n_tokens) {
        int e;
        float w;
        choose(p, sh.correction, sh.bias, z + warp * z_row, keys + warp * (p.n_out + p.n_groups), lane, e, w);
        const bool have = lane < p.top, real = have && e < p.n_real;
        const float identity = warp_sum(have && !real ? w : 0.f);
        if (real) {
            atomicOr(&sh.tokens[e], 1u << warp);
            atomicOr(&sh.choice[e], (unsigned long long)lane << (4 * warp));
        }
        if (lane == 0) {
            sh.gate[warp] = p.shared_gate ? logistic(z[warp * z_row + p.n_out]) : 1.f;
            sh.plan.identity[warp] = identity;
        }
        __syncwarp();
        if (real) z[warp * z_row + e] = w;
    }
    __syncthreads();
    // the experts that some token chose, ascending: every warp counts them all, 32 at a vote, and writes down its own
    int n_active = 0, n_work = 0;
    for (int c = 0; c * 32 < p.n_real; ++c) {
        const int e = c * 32 + lane;
        const unsigned tokens = e < p.n_real ? sh.tokens[e] : 0u, votes = __ballot_sync(0xffffffffu, tokens != 0u), below = (1u << lane) - 1u;
        const unsigned many = __ballot_sync(0xffffffffu, __popc(tokens) > 8);
        if (warp == c % L_WARPS && tokens != 0u) {
            const int at = n_active + __popc(votes & below), w = n_work + __popc(votes & below) + __popc(many & below);
            ActiveExpert& a = sh.plan.of[at];
            unsigned long long list = 0ull;
            int n = 0;
            for (unsigned m = tokens; m != 0u; m &= m - 1u, ++n) list |= (unsigned long long)(__ffs((int)m) - 1) << (4 * n);
            a.expert = e;
            a.tokens = tokens;
            a.list = list;
            a.choice = sh.choice[e];
            sh.work[w] = (unsigned short)at;
            if (n > 8) sh.work[w + 1] = (unsigned short)((unsigned)at | SECOND);
        }
        n_active += __popc(votes);
        n_work += __popc(votes) + __popc(many);
    }
    if (threadIdx.x == 0) sh.plan.n_active = n_active;
    __syncthreads();
    if (blockIdx.x == 0) {
        const int words = (int)(offsetof(LayerPlan, of) + (size_t)n_active * sizeof(ActiveExpert)) / 8;
        for (int i = threadIdx.x; i < words; i += L_THREADS) reinterpret_cast<unsigned long long*>(p.plan)[i] = reinterpret_cast<const unsigned long long*>(&sh.plan)[i];
    }
    pdl_trigger();

    // items: eight features for up to eight tokens, of the shared expert, then of the active ones; a team's warp takes every TEAM-th chunk of their k, a round each
    const int per_shared = p.inner_shared / 8, shared_items = per_shared * ((p.n_tokens + 7) / 8), per_expert = p.inner / 8, n_items = shared_items + n_work * per_expert;
    const int n_chunks = (p.width + LK - 1) / LK, rounds = (n_chunks + TEAM - 1) / TEAM;
    const int team = warp / TEAM, member = warp % TEAM, stride = gridDim.x * TEAMS, first = team * gridDim.x + blockIdx.x;
    struct Item {
        bool own, second;           // not the shared expert's; after the first eight tokens
        int a, f0;                  // which active expert's, from which feature on
    };
    auto item_of = [&](int item) {
        Item it;
        it.own = item >= shared_items;
        const int w = it.own ? quotient(item - shared_items, p.per_expert_magic) : 0, entry = it.own ? sh.work[w] : 0;
        it.second = it.own ? (entry & SECOND) != 0u : item >= per_shared;
        it.a = entry & (SECOND - 1u);
        it.f0 = (it.own ? item - shared_items - w * per_expert : it.second ? item - per_shared : item) * 8;
        return it;
    };
    // an item's rows and their scales: row g of the 16 is a gate row, row g + 8 the row of the linear branch of the same feature
    const unsigned char *row0 = nullptr, *row1 = nullptr;
    const float *scale0 = nullptr, *scale1 = nullptr;
    auto rows_of = [&](int item) {
        const Item it = item_of(item);
        const int f = it.f0 + g, e = it.own ? sh.plan.of[it.a].expert : 0;
        const LayerMatrix& m = it.own ? p.up : p.shared_up;
        const int il = it.own ? p.interleave : p.interleave_shared;
        const int r0 = il == 0 ? f : il == 4 ? 2 * f - (f & 3) : f / il * 2 * il + f % il, r1 = r0 + (il > 0 ? il : it.own ? p.inner : p.inner_shared);
        const unsigned char* base = m.w + e * m.stack_bytes;
        row0 = base + r0 * m.row_bytes;
        row1 = base + r1 * m.row_bytes;
        if (CODES) {
            const float* scales = m.scales + (long long)e * m.row_blocks * m.k_blocks;
            scale0 = scales + (long long)(r0 / LK) * m.k_blocks;
            scale1 = scales + (long long)(r1 / LK) * m.k_blocks;
        }
    };
    // A chunk of bfloat16 and the next one in turn, one on its way while the other is worked on; or two chunks of codes at once.  (Two pairs of codes, or three or four
    // chunks in turn: 50.9, 57.1 and 53.6 us instead of 48.3 for 8 tokens and 20 experts of 1,024: more code to fetch.)
    constexpr int UNIT = CODES ? 2 : 1, UNITS = CODES ? 1 : 2, TURN = UNITS * UNIT;
    const int turns = (rounds + TURN - 1) / TURN * TURN;
    Chunk<CODES> held[UNITS][UNIT];
    auto load = [&](Chunk<CODES> (&unit)[UNIT], int round) {
#pragma unroll
        for (int i = 0; i < UNIT; ++i) {
            const int chunk = min(member + (round + i) * TEAM, n_chunks - 1);
            load_chunk<CODES>(unit[i], row0, row1, chunk * LK, p.width, lane);
            if (CODES) unit[i].scale[0] = scale0[chunk], unit[i].scale[1] = scale1[chunk];
        }
    };
    if (first < n_items) {
        rows_of(first);
#pragma unroll
        for (int u = 0; u < UNITS; ++u) load(held[u], u * UNIT);
    }
    int set = 0;
#pragma unroll 1
    for (int item = first; item < n_items; item += stride) {
        {
            // this lane's column: a token that chose the expert, or any for the shared one (behind them token 0, whose sums nobody reads)
            const Item it = item_of(item);
            const unsigned long long every = it.own ? sh.plan.of[it.a].list : 0xfedcba9876543210ull;
            const unsigned list = (unsigned)(it.second ? every >> 32 : every);
            const int n_cols = min(8, (it.own ? __popc(sh.plan.of[it.a].tokens) : p.n_tokens) - (it.second ? 8 : 0)), token = (int)(list >> (4 * g)) & 15;
            const bf16* x = x_copy + (long long)(g < n_cols ? token : 0) * p.x_row + (lane & 3) * (CODES ? 16 : 8) + member * LK;
            float acc[4] = {};
#pragma unroll 1
            for (int round = 0; round < turns; round += TURN) {
                const bool last = round + TURN >= turns, more = !last || item + stride < n_items;
                if (last && more) rows_of(item + stride);
#pragma unroll
                for (int u = 0; u < UNITS; ++u, x += UNIT * TEAM * LK) {
                    if (member + (round + u * UNIT) * TEAM < n_chunks) {
                        // (a unit's second chunk that is not there is the last one again and meets zeros)
                        Column<CODES> columns[UNIT];
#pragma unroll
                        for (int i = 0; i < UNIT; ++i) load_column<CODES>(columns[i], x + i * TEAM * LK);
#pragma unroll
                        for (int i = 0; i < UNIT; ++i) multiply<CODES>(held[u][i], columns[i], acc);
                    }
                    if (more) load(held[u], last ? u * UNIT : round + TURN + u * UNIT);
                }
            }
            auto& mine = sh.reduce[set][warp];
            const int col = (lane & 3) * 2;
            mine[g][col] = acc[0];
            mine[g][col + 1] = acc[1];
            mine[g + 8][col] = acc[2];
            mine[g + 8][col + 1] = acc[3];
            // The team's warps take the ends of items in turn, and the others go on.  (As many sets as warps: before a warp writes a set again it has ended an item
            // itself since, for which it waited for all; the warp that read the set had done so by then.)  Barriers 0 .. 15: nothing else uses one from here on.
            const int barrier = team * TEAM + set, mine_to_end = set == member;
            set = set + 1 == TEAM ? 0 : set + 1;
            if (!mine_to_end) {
                asm volatile("bar.arrive %0, %1;" ::"r"(barrier), "n"(32 * TEAM) : "memory");
                continue;
            }
            asm volatile("bar.sync %0, %1;" ::"r"(barrier), "n"(32 * TEAM) : "memory");
            const int f = lane & 7;
#pragma unroll 1
            for (int c = lane >> 3; c < n_cols; c += 4) {
                float gate = 0.f, lin = 0.f;
#pragma unroll
                for (int w = 0; w < TEAM; ++w) {
                    gate += sh.reduce[member][team * TEAM + w][f][c];
                    lin += sh.reduce[member][team * TEAM + w][f + 8][c];
                }
                const int t = (int)(list >> (4 * c)) & 15;
                const ActiveExpert& ex = sh.plan.of[it.a];
                const int row = it.own ? t * p.top + ((int)(ex.choice >> (4 * t)) & 15) : p.n_tokens * p.top + t;
                const float w = it.own ? z[t * z_row + ex.expert] : sh.gate[t];
                if (CODES) {
                    const float back = unscaling_of(sh.exponent[t]);
                    gate *= back;
                    lin *= back;
                }
                if (p.limit != INFINITY) {          // (a NaN stays one)
                    gate = gate > p.limit ? p.limit : gate;
                    lin = lin > p.limit ? p.limit : lin < -p.limit ? -p.limit : lin;
                }
                const float v = glu_gate(gate, p.slope) * (lin + p.shift) * w;
                const long long at = (long long)row * p.h_row + it.f0 + f;
                if (CODES) {
                    p.h[at] = v;
                } else {
                    bf16 hi = __float2bfloat16_rn(v);
                    if (__hisinf(hi)) hi = __float2bfloat16_rz(v);          // (beyond the largest bfloat16 the second number makes up for it)
                    p.h_hi[at] = hi;
                    p.h_lo[at] = __float2bfloat16_rn(v - __bfloat162float(hi));
                }
            }
        }
    }
}

// ---- down ------------------------------------------------------------------------------------------------------------------------------

constexpr int PARTS = 4;                                    // CTAs of a cluster: they share the chunks
constexpr int LEAST_TEAMS = 2, MOST_TEAMS = 4;              // of a CTA: each has 16 output features of its own, and its warps share the CTA's chunks
constexpr int HELD = 2;                                     // chunks that a warp has on their way
constexpr int SLOT = LK * 4;                                // bytes of a piece: its first numbers, and behind them the second ones

struct DownShared {
    float reduce[L_WARPS][16][LT + 1];
    float sums[2][PARTS][16][LT];                           // of the CTAs' teams, for the CTA that ends their features (in turn)
    LayerPlan plan;
    int n_slots, next;                                      // of h's pieces that are in shared memory, and the first chunk whose are not
};
// Behind it, for `cap` slots: h's pieces (128 k of a token's row), then what brings a slot's sums back, where a slot's piece lies in h (row * 128 + chunk of its k),
// and the first slot of a chunk.
constexpr size_t down_smem_bytes(int cap) { return sizeof(DownShared) + (size_t)cap * (SLOT + 4 + 2 + 2); }
// What a CTA takes of shared memory at most: the rest is the first-level cache, through which the weights on their way go (16 tokens, 50 experts of 1,408 of width 2,048
// and a shared one, in bfloat16, whose pieces would fill it: 353, 214 and 179 us with 227, 195 and 163 KB, the pieces in one, two and two goes).
constexpr int DOWN_SMEM = 163 * 1024;
constexpr int MOST_SLOTS = (int)((DOWN_SMEM - sizeof(DownShared)) / (SLOT + 8)) / 8 * 8;
static_assert(MOST_TEAMS <= PARTS && L_THREADS == 512, "a CTA for each team's end");
static_assert(sizeof(DownShared) % 16 == 0, "vectors of 16 bytes behind it");
static_assert(MOST_SLOTS >= LT * L_WARPS / LEAST_TEAMS * HELD, "a turn of all warps' chunks with all tokens");
static_assert((L_MAX_PAIRS + LT) * (MOST_K / LK) <= 65536, "a piece's place in 16 bits");

// Where unit u of eight k lies within a slot: the four lanes of a load side by side (beside codes a lane takes 16 k, two units, at a time), the halves of odd slots
// exchanged, so that the two slots that a quarter of a warp reads meet in no bank.
template <bool CODES> __device__ __forceinline__ int unit_of(int u, int slot) {
    const int at = CODES ? (u & 8) | (u & 1) << 2 | (u >> 1 & 3) : u;
    return at ^ (slot & 1) << 2;
}

// The sum of the products with h's first numbers and of those with the second: where the first is infinite, by an h or a weight that is, the second says nothing.
__device__ __forceinline__ float joined(float first, float second) { return fabsf(first) < INFINITY ? first + second : first; }

// A cluster takes 16 * teams output features at a time; the chunks (of the shared expert, then of the active ones) go round its CTAs, and round the warps of a
// team.
template <bool CODES, int GROUPS>
__global__ __launch_bounds__(L_THREADS, 1) void moe_layer_down_kernel(const LayerArgs p, int teams, int cap) {
    extern __shared__ __align__(16) unsigned char down_smem[];
    DownShared& sh = *reinterpret_cast<DownShared*>(down_smem);
    unsigned char* pieces = down_smem + sizeof(DownShared);
    float* back = reinterpret_cast<float*>(pieces + (size_t)cap * SLOT);
    unsigned short *place = reinterpret_cast<unsigned short*>(back + cap), *slot_of = place + cap;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2;
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    const int rank = blockIdx.x % PARTS, n_groups = (p.width + 15) / 16, clusters = gridDim.x / PARTS;
    const int members = L_WARPS / teams, team = warp / members, member = warp % members;
    // this CTA's chunks: number i is chunk rank + PARTS * i of all, those of the shared expert first (until the plan is known, all)
    const int own_chunks = (p.inner + LK - 1) / LK, shared_chunks = (p.inner_shared + LK - 1) / LK;
    int n_chunks = (shared_chunks - rank + PARTS - 1) / PARTS;
    struct Place {              // a chunk: which active expert's (or the shared one's), and where in its k
        bool own;
        int a, kb;
        unsigned tokens;
    };
    auto place_of = [&](int i) {
        const int chunk = rank + PARTS * i;
        Place at;
        at.own = chunk >= shared_chunks;
        at.a = at.own ? quotient(chunk - shared_chunks, p.own_chunks_magic) : 0;
        at.kb = at.own ? (chunk - shared_chunks) - at.a * own_chunks : chunk;
        at.tokens = at.own ? sh.plan.of[at.a].tokens : (1u << p.n_tokens) - 1u;
        return at;
    };
    auto load = [&](Chunk<CODES>& c, int group, int i) {
        if (i >= n_chunks) return;
        const Place at = place_of(i);
        const LayerMatrix& m = at.own ? p.down : p.shared_down;
        const int e = at.own ? sh.plan.of[at.a].expert : 0, r0 = min(group * 16 + g, p.width - 1), r1 = min(group * 16 + g + 8, p.width - 1);
        const unsigned char* base = m.w + e * m.stack_bytes;
        load_chunk<CODES>(c, base + r0 * m.row_bytes, base + r1 * m.row_bytes, at.kb * LK, at.own ? p.inner : p.inner_shared, lane);
        if (CODES)      // (sixteen rows lie in one block)
            c.scale[0] = m.scales[((long long)e * m.row_blocks + r0 / LK) * m.k_blocks + at.kb];
    };
    // The pieces of h that the chunks from `from` on meet, as many as there are slots for (whole turns of all warps), into shared memory; beside codes scaled.
    auto fill = [&](int from) {
        __syncthreads();                // nobody reads the last ones any more
        if (warp == 0) {
            int used = 0, i = from;
            for (bool room = true; room && i < n_chunks;) {
                const bool have = i + lane < n_chunks;
                const Place at = place_of(have ? i + lane : from);
                const int n = have ? __popc(at.tokens) : 0;
                int upto = n;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int v = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += v;
                }
                const unsigned fits = __ballot_sync(0xffffffffu, have && used + upto <= cap);
                int take = __popc(fits);
                if (take < min(32, n_chunks - i)) {
                    room = false;
                    take -= (i + take - from) % (members * HELD);           // (no less than none: see the assertion above)
                }
                const int first = used + upto - n;
                if (lane < take) {
                    slot_of[i + lane - from] = (unsigned short)first;
                    int k = first;
                    for (unsigned m = at.tokens; m != 0u; m &= m - 1u, ++k) {
                        const int t = __ffs((int)m) - 1;
                        const int row = at.own ? t * p.top + ((int)(sh.plan.of[at.a].choice >> (4 * t)) & 15) : p.n_tokens * p.top + t;
                        place[k] = (unsigned short)(row * (MOST_K / LK) + at.kb);
                    }
                }
                used = take > 0 ? __shfl_sync(0xffffffffu, used + upto, take - 1) : used;
                i += take;
            }
            if (lane == 0) {
                sh.n_slots = used;
                sh.next = i;
            }
        }
        __syncthreads();
        // (the loads of several slots are asked for before the first is used: they come from the second-level cache)
        const int n_slots = sh.n_slots;
        constexpr int AT_ONCE = 6;
        for (int slot0 = warp; slot0 < n_slots; slot0 += AT_ONCE * L_WARPS) {
            uint4 v[AT_ONCE];
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                const int slot = slot0 + i * L_WARPS, at = slot < n_slots ? place[slot] : 0;
                const int row = at / (MOST_K / LK), inner = row < p.n_tokens * p.top ? p.inner : p.inner_shared;
                const int k = at % (MOST_K / LK) * LK + (CODES ? lane * 4 : (lane & 15) * 8);
                const long long from = (long long)row * p.h_row + k;
                v[i] = make_uint4(0, 0, 0, 0);
                if (slot < n_slots && k < inner)
                    v[i] = CODES ? *reinterpret_cast<const uint4*>(p.h + from) : *reinterpret_cast<const uint4*>((lane < 16 ? p.h_hi : p.h_lo) + from);
            }
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                const int slot = slot0 + i * L_WARPS;
                if (slot >= n_slots) break;
                unsigned char* to = pieces + (size_t)slot * SLOT;
                if constexpr (CODES) {
                    const unsigned top = max(max(v[i].x & 0x7fffffffu, v[i].y & 0x7fffffffu), max(v[i].z & 0x7fffffffu, v[i].w & 0x7fffffffu));
                    const int e = max((int)(__reduce_max_sync(0xffffffffu, top) >> 23), LEAST_EXPONENT);
                    const float scaling = scaling_of(e);
                    uint2 hi, lo;
                    split_half(__uint_as_float(v[i].x) * scaling, __uint_as_float(v[i].y) * scaling, hi.x, lo.x);
                    split_half(__uint_as_float(v[i].z) * scaling, __uint_as_float(v[i].w) * scaling, hi.y, lo.y);
                    to += unit_of<CODES>(lane >> 1, slot) * 16 + (lane & 1) * 8;
                    *reinterpret_cast<uint2*>(to) = hi;
                    *reinterpret_cast<uint2*>(to + LK * 2) = lo;
                    if (lane == 0) back[slot] = unscaling_of(e);
                } else {
                    *reinterpret_cast<uint4*>(to + (lane >> 4) * (LK * 2) + unit_of<CODES>(lane & 15, slot) * 16) = v[i];
                }
            }
        }
        __syncthreads();
    };

    Chunk<CODES> held[HELD];
    int group = (blockIdx.x / PARTS) * teams + team;
    // The first chunks: those of the shared expert before the up kernel has finished (its CTAs have waited for what came before, so nobody writes a weight any more),
    // the others when the plan is there.
#pragma unroll 1
    for (int known = 0, planned = 0;; planned = 1) {
#pragma unroll
        for (int u = 0; u < HELD; ++u)
            if (member + u * members >= known) load(held[u], group, member + u * members);
        if (planned) break;
        pdl_wait();
        // (as much of the plan as the step can have: its length comes with it)
        const int words = (int)(offsetof(LayerPlan, of) + (size_t)min(p.n_tokens * p.top, p.n_real) * sizeof(ActiveExpert)) / 8;
        for (int i = threadIdx.x; i < words; i += L_THREADS) reinterpret_cast<unsigned long long*>(&sh.plan)[i] = reinterpret_cast<const unsigned long long*>(p.plan)[i];
        __syncthreads();
        pdl_trigger();
        known = n_chunks;
        n_chunks = (shared_chunks + sh.plan.n_active * own_chunks - rank + PARTS - 1) / PARTS;
    }
    // every CTA of the cluster has begun before its shared memory is written from another
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    int set = 0, from = 0, upto = 0;    // the chunks whose pieces are in shared memory: all of them, as a rule
#pragma unroll 1
    for (int group0 = group - team; group0 < n_groups; group0 += clusters * teams, group += clusters * teams) {
        float acc[GROUPS][4] = {};
#pragma unroll 1
        for (int turn = 0; turn < n_chunks; turn += HELD * members) {
            if (turn < from || turn >= upto) {
                fill(turn);
                from = turn;
                upto = sh.next;
            }
#pragma unroll
            for (int u = 0; u < HELD; ++u) {
                const int i = turn + u * members + member;
                if (i < n_chunks) {
                    const Place at = place_of(i);
                    const int first = slot_of[i - from];
                    uint32_t a[Chunk<CODES>::STEPS][Chunk<CODES>::PARTS][4];
#pragma unroll
                    for (int s = 0; s < Chunk<CODES>::STEPS; ++s)
#pragma unroll
                        for (int j = 0; j < Chunk<CODES>::PARTS; ++j) held[u].operand(s, j, a[s][j]);
                    const float scale = CODES ? held[u].scale[0] : 1.f;
                    constexpr int VECS = Column<CODES>::VECS;
#pragma unroll
                    for (int n = 0; n < GROUPS; ++n) {
                        if (GROUPS > 1 && (at.tokens >> (8 * n) & 0xffu) == 0u) continue;
                        // the columns: the tokens that chose the chunk's expert (the others': any of them; their sums are left out, so that a weight that is no
                        // number does not reach them)
                        const int t = n * 8 + g, slot = first + (at.tokens >> t & 1u ? __popc(at.tokens & ((1u << t) - 1u)) : 0);
                        const unsigned char* piece = pieces + (size_t)slot * SLOT;
                        const int flip = (slot & 1) << 6;
                        float part[2][4] = {};
#pragma unroll
                        for (int s = 0; s < Chunk<CODES>::STEPS; ++s) {
#pragma unroll
                            for (int v = 0; v < VECS; ++v) {        // (codes: the halves of the step's k)
                                const unsigned char* at_k = piece + ((s * VECS + v) * 64 + (lane & 3) * 16 ^ flip);
                                const uint4 b = *reinterpret_cast<const uint4*>(at_k), c = *reinterpret_cast<const uint4*>(at_k + LK * 2);
#pragma unroll
                                for (int j = 0; j < 2; ++j) {       // h's two numbers in turn
                                    mma_step<CODES>(part[0], a[s][2 * v + j], j ? b.z : b.x, j ? b.w : b.y);
                                    mma_step<CODES>(part[1], a[s][2 * v + j], j ? c.z : c.x, j ? c.w : c.y);
                                }
                            }
                        }
                        const int t0 = n * 8 + (lane & 3) * 2;
#pragma unroll
                        for (int c = 0; c < 2; ++c)
                            if (at.tokens >> (t0 + c) & 1u) {
                                // (of the two scales the large one first meets the small one, so that a sum leaves float32's range only if the result does)
                                const float by = CODES ? back[first + __popc(at.tokens & ((1u << (t0 + c)) - 1u))] : 1.f;
                                const float one = by > 1.f ? by * scale : by, two = by > 1.f ? 1.f : scale;
                                acc[n][c] = fmaf(joined(part[0][c], part[1][c]) * one, two, acc[n][c]);
                                acc[n][2 + c] = fmaf(joined(part[0][2 + c], part[1][2 + c]) * one, two, acc[n][2 + c]);
                            }
                    }
                }
                if (turn + HELD * members < n_chunks) load(held[u], group, i + HELD * members);
                else if (group0 + clusters * teams < n_groups) load(held[u], group + clusters * teams, member + u * members);
            }
        }
        const int col = (lane & 3) * 2;
#pragma unroll
        for (int n = 0; n < GROUPS; ++n) {
            sh.reduce[warp][g][n * 8 + col] = acc[n][0];
            sh.reduce[warp][g][n * 8 + col + 1] = acc[n][1];
            sh.reduce[warp][g + 8][n * 8 + col] = acc[n][2];
            sh.reduce[warp][g + 8][n * 8 + col + 1] = acc[n][3];
        }
        __syncthreads();
        // CTA r ends the features of team r: every CTA adds its team's sums in order and hands them over, and CTA r adds the four.  (Two sets: a CTA writes one again
        // after the next meeting, to which everybody comes when they have read it.)
        const int f = threadIdx.x & 15, t = threadIdx.x >> 4 & 15;
        for (int to = threadIdx.x >> 8; to < teams; to += 2) {
            float v = 0.f;
            for (int m = 0; m < members; ++m) v += sh.reduce[to * members + m][f][t];
            st_cluster_f32(&sh.sums[set][rank][f][t], v, (uint32_t)to);
        }
        cluster_sync_all();
        const int feature = (group0 + rank) * 16 + f;
        if (threadIdx.x < 256 && rank < teams && t < p.n_tokens && feature < p.width) {
            float v = 0.f;
#pragma unroll
            for (int r = 0; r < PARTS; ++r) v += sh.sums[set][r][f][t];
            const float w = sh.plan.identity[t];
            if (p.n_out > p.n_real) v += w * __bfloat162float(p.x[(long long)t * p.ldx + feature]);
            p.out[(long long)t * p.width + feature] = __float2bfloat16_rn(v);
        }
        set ^= 1;
    }
}

template <int GROUPS, int TEAM> size_t up_smem_bytes(const LayerArgs& p) { return sizeof(UpShared<GROUPS, TEAM>) + (size_t)LT * (p.n_out + 1) * 4 + (size_t)LT * (p.n_out + p.n_groups) * 4; }

// Clusters of `size` CTAs that the device holds at once, one CTA to an SM (asked for once a device): the clusters of a grid that come in a second round begin when the
// others are done.
template <typename... KArgs> int clusters_at_once(void (*kernel)(KArgs...), int size, size_t smem, int sms, std::atomic<int> (&known)[64]) {
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 1;
    if (dev < 64 && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(64 * size);
    cfg.blockDim = dim3(L_THREADS);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) n = 1;
    if (n > sms / size) n = sms / size > 0 ? sms / size : 1;            // (what the workspace has room for)
    if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
    return n;
}

template <bool CODES, int GROUPS, int TEAM> int launch_layer(const LayerArgs& p, int sms, cudaStream_t stream) {
    static std::atomic<unsigned long long> allowed_up{0}, allowed_down{0};
    static std::atomic<int> known_up[64], known_down[64];
    static_assert(sizeof(UpShared<GROUPS, TEAM>) + (size_t)LT * (L_MAX_OUT + 1) * 4 + (size_t)LT * 2 * L_MAX_OUT * 4 <= 227 * 1024, "the most router outputs and groups");
    cudaError_t e = rlis_allow_smem(moe_layer_up_kernel<CODES, GROUPS, TEAM>, 227 * 1024, allowed_up);
    if (e == cudaSuccess) e = rlis_allow_smem(moe_layer_down_kernel<CODES, GROUPS>, DOWN_SMEM, allowed_down);
    if (e != cudaSuccess) return (int)e;
    const size_t up_smem = up_smem_bytes<GROUPS, TEAM>(p);
    const int up_clusters = clusters_at_once(moe_layer_up_kernel<CODES, GROUPS, TEAM>, L_CLUSTER, up_smem, sms, known_up);
    rlis_launch_cluster(moe_layer_up_kernel<CODES, GROUPS, TEAM>, dim3((unsigned)(up_clusters * L_CLUSTER)), dim3(L_THREADS), up_smem, stream, dim3(L_CLUSTER, 1, 1), p);
    const int rc = RLIS_LAUNCH_CHECK();
    if (rc != 0) return rc;
    // as many slots as the pieces of a CTA's chunks can take, up to what its shared memory holds
    const auto share = [](int k) { return ((k + LK - 1) / LK + PARTS - 1) / PARTS; };
    const int all = p.n_tokens * (p.top * share(p.inner) + share(p.inner_shared)), cap = all < MOST_SLOTS ? (all + 7) / 8 * 8 : MOST_SLOTS;
    const int groups = (p.width + 15) / 16;
    const int teams = (groups + MOST_TEAMS - 1) / MOST_TEAMS * PARTS * 4 >= 3 * sms ? MOST_TEAMS : LEAST_TEAMS;
    const int most = clusters_at_once(moe_layer_down_kernel<CODES, GROUPS>, PARTS, down_smem_bytes(MOST_SLOTS), sms, known_down);
    const int clusters = (groups + teams - 1) / teams < most ? (groups + teams - 1) / teams : most;
    rlis_launch_cluster(moe_layer_down_kernel<CODES, GROUPS>, dim3((unsigned)(clusters * PARTS)), dim3(L_THREADS), down_smem_bytes(cap), stream, dim3(PARTS, 1, 1), p,
                        teams, cap);
    return RLIS_LAUNCH_CHECK();
}
}  // namespace

// What a matrix of the layer is, as the host hands it over: rows row_bytes and the matrices of a stack stack_bytes apart; scales null: bfloat16, else codes.
struct RlisLayerMatrix {
    const void* w;
    const float* scales;
    long long row_bytes, stack_bytes;
};
struct RlisMoeLayer {
    const void* x;
    long long ldx;
    const float *router, *correction, *router_bias;
    RlisLayerMatrix up, down, shared_up, shared_down;
    void *workspace, *out;
    int n_tokens, width, inner, inner_shared, n_experts, n_identity, top, scoring, n_groups, keep_groups, normalize, shared_gate, interleave, interleave_shared;
    float route_scale, slope, limit, shift;
};

namespace {
// Where a call's parts of the workspace lie; `bytes` of it in all.
struct LayerSpace {
    long long h, x, bytes;
    int h_row, x_row;
};
LayerSpace space_of(int n_tokens, int top, int width, int inner, int inner_shared, int sms) {
    LayerSpace s;
    const long long rows = (long long)n_tokens * (top + 1);
    s.h_row = inner > inner_shared ? inner : inner_shared;
    s.x_row = (width + LK - 1) / LK * LK + MOST_TEAM * LK;     // (a chunk more for a team's second chunks)
    s.h = (sizeof(LayerPlan) + 15) / 16 * 16;
    s.x = s.h + 4 * rows * s.h_row;
    s.bytes = s.x + (long long)(sms / L_CLUSTER + 1) * n_tokens * s.x_row * 2;
    return s;
}
int layer_sms() {
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms;
}
}  // namespace

// Bytes of workspace of a call on the current device (0: a size that is not taken).
extern "C" long long rlis_moe_layer_bytes(int n_tokens, int top, int width, int inner, int inner_shared) {
    if (n_tokens < 0 || n_tokens > LT || top < 0 || top > L_MAX_PAIRS / LT || width < 0 || inner < 0 || inner_shared < 0) return 0;
    return space_of(n_tokens, top, width, inner, inner_shared, layer_sms()).bytes;
}

extern "C" int rlis_moe_layer(const RlisMoeLayer* a, cudaStream_t stream) {
    if (a->n_tokens <= 0) return 0;
    const int n_out = a->n_experts + a->n_identity;
    const bool codes = a->up.scales != nullptr, shared = a->inner_shared > 0;
    const int unit = codes ? 16 : 8;                // k in 16 bytes
    if (a->n_tokens > LT || a->n_experts <= 0 || a->n_identity < 0 || n_out > L_MAX_OUT || a->top <= 0 || a->top > n_out || a->top > L_MAX_PAIRS / LT || a->scoring < 0 ||
        a->scoring > 2 || a->n_groups < 1 || n_out % a->n_groups != 0 || a->keep_groups < 1 || a->keep_groups > a->n_groups ||
        a->top > a->keep_groups * (n_out / a->n_groups) || a->width <= 0 || a->width % unit != 0 || a->inner <= 0 || a->inner % unit != 0 || a->inner_shared % unit != 0 ||
        a->inner_shared < 0 || (a->shared_gate && !shared) || a->interleave < 0 || (a->interleave > 0 && a->inner % a->interleave != 0) || a->interleave_shared < 0 ||
        (a->interleave_shared > 0 && a->inner_shared % a->interleave_shared != 0) || a->width > MOST_K || a->inner > MOST_K || a->inner_shared > MOST_K)
        return RLIS_ERR_UNSUPPORTED;
    // (every lane has the scales of its own rows, so any interleaving would do; beside codes groups of fewer than four rows are not offered, since no loader lays them out)
    if (codes && (a->interleave % 4 != 0 || a->interleave_shared % 4 != 0)) return RLIS_ERR_UNSUPPORTED;
    if ((reinterpret_cast<uintptr_t>(a->x) & 15) != 0 || a->ldx % 8 != 0 || (reinterpret_cast<uintptr_t>(a->router) & 15) != 0 || (reinterpret_cast<uintptr_t>(a->workspace) & 15) != 0)
        return RLIS_ERR_UNSUPPORTED;
    const RlisLayerMatrix* all[4] = {&a->up, &a->down, &a->shared_up, &a->shared_down};
    for (int i = 0; i < (shared ? 4 : 2); ++i)
        if ((reinterpret_cast<uintptr_t>(all[i]->w) & 15) != 0 || all[i]->row_bytes % 16 != 0 || all[i]->stack_bytes % 16 != 0 || (all[i]->scales != nullptr) != codes)
            return RLIS_ERR_UNSUPPORTED;
    LayerArgs p{};
    p.x = static_cast<const bf16*>(a->x);
    p.ldx = a->ldx;
    p.n_tokens = a->n_tokens;
    p.width = a->width;
    p.router = a->router;
    p.correction = a->correction;
    p.router_bias = a->router_bias;
    p.n_out = n_out;
    p.n_real = a->n_experts;
    p.top = a->top;
    p.scoring = a->scoring;
    p.n_groups = a->n_groups;
    p.keep_groups = a->keep_groups;
    p.normalize = a->normalize;
    p.shared_gate = a->shared_gate ? 1 : 0;
    p.route_scale = a->route_scale;
    p.inner = a->inner;
    p.inner_shared = a->inner_shared;
    p.interleave = a->interleave;
    p.interleave_shared = a->interleave_shared;
    auto matrix = [](const RlisLayerMatrix& m, int rows, int k) {
        return LayerMatrix{static_cast<const unsigned char*>(m.w), m.scales, m.row_bytes, m.stack_bytes, (rows + LK - 1) / LK, (k + LK - 1) / LK};
    };
    p.up = matrix(a->up, 2 * a->inner, a->width);
    p.down = matrix(a->down, a->width, a->inner);
    p.shared_up = matrix(a->shared_up, 2 * a->inner_shared, a->width);
    p.shared_down = matrix(a->shared_down, a->width, a->inner_shared);
    p.slope = a->slope;
    p.limit = a->limit;
    p.shift = a->shift;
    p.plan = static_cast<LayerPlan*>(a->workspace);
    const int sms = layer_sms();
    const LayerSpace space = space_of(a->n_tokens, a->top, a->width, a->inner, a->inner_shared, sms);
    unsigned char* work = static_cast<unsigned char*>(a->workspace);
    p.h_row = space.h_row;
    p.h_hi = reinterpret_cast<bf16*>(work + space.h);
    p.h_lo = p.h_hi + (long long)a->n_tokens * (a->top + 1) * p.h_row;
    p.h = reinterpret_cast<float*>(work + space.h);
    p.x_copy = reinterpret_cast<bf16*>(work + space.x);
    p.x_row = space.x_row;
    p.out = static_cast<bf16*>(a->out);
    auto magic = [](int d) { return d > 1 ? (unsigned)(((1ull << 32) + d - 1) / d) : 0u; };
    p.per_expert_magic = magic(a->inner / 8);
    p.own_chunks_magic = magic((a->inner + LK - 1) / LK);
    // Where teams of four warps would take two items each at the most, many would take one while others take two: teams of eight take twice as many half as long ones,
    // as long as a warp has two chunks of each (one token, 4 of 32 experts of 1,024 of width 2,048 and a shared one: 25.5 -> 24.2 us, in blocks 21.3 -> 20.8; 8 tokens, 22
    // experts: 63.6 -> 62.8, but in blocks 46.4 -> 50.1).
    const int items = (p.n_tokens * p.top * p.inner + p.inner_shared) / 8, teams = sms / L_CLUSTER * L_CLUSTER * (L_WARPS / 4);
    if (p.n_tokens <= 8 && items <= 2 * teams && p.width > 15 * LK) return codes ? launch_layer<true, 1, 8>(p, sms, stream) : launch_layer<false, 1, 8>(p, sms, stream);
    if (p.n_tokens <= 8) return codes ? launch_layer<true, 1, 4>(p, sms, stream) : launch_layer<false, 1, 4>(p, sms, stream);
    return codes ? launch_layer<true, 2, 4>(p, sms, stream) : launch_layer<false, 2, 4>(p, sms, stream);
}
