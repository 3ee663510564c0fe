// A whole mixture of experts for up to 16 tokens in two kernels (moe.cu says what each part of it computes):
//
//   up:   z = W_r x, the choice of `top` outputs a token and their weights; h[t, e, :] = weight[t, e] glu(W_gate_e x_t, W_up_e x_t) for the chosen pairs, and
//         h[t, s, :] = gate[t] glu(..) of the shared expert
//   down: out[t, :] = sum over e of W_down_e h[t, e, :] (+ W_down_s h[t, s, :]) + sum of the weights of t's identity experts * x_t
//
// With so few tokens the layer is a stream of the chosen experts' weights from memory (8 tokens, 4 of 32 experts of 2,048 x 1,024 and a shared one: 278 MB, 42 us
// at the rate of a copy).  So every weight is read once, by 16-byte loads of 16 rows side by side straight into the registers of mma.sync m16n8k16, no
// shared memory between: a sum over k may take k in any order, so a thread's 16 bytes of a row, eight neighbouring k, serve as its k slots of two
// instructions, and the tokens' rows, which stay in the first-level cache, are read in the same order.  A warp takes 128 k of 16 rows at a time (a chunk, a
// block's edge; for weights in e4m3 blocks a chunk's sums are scaled before they join the others) and has the next chunks, of the next rows if need be, on
// their way while it works on one: 128 KB an SM (96 KB of codes) are in flight.  Four warps (up) or a CTA's sixteen (down) take different k of the same rows
// and add their sums in shared memory in the order of the warps, so results do not depend on timing.
//
// Routing sits in the up kernel: the CTAs of a cluster share the router's rows, hand each other the logits (distributed shared memory), and each chooses
// for all tokens itself: no launch of its own, no grid-wide barrier, no workspace but h and the plan, which the first CTA leaves for the down kernel.  The
// router's float32 rows go through the same instructions as three bfloat16 numbers each, whose sum they are to 2^-24 (a token's logits are sums of exact
// products in float32, as a chain of FMAs would give them; as FMAs, 128 rows against 16 tokens took 20 us).
//
// The weights of the choice are multiplied into h in float32, and h is handed on as two bfloat16 numbers (their sum is h to 2^-17), so that nothing but the
// result is rounded to the activations' type; the down product is then one long sum over the chosen experts' k, with the step's tokens as columns whoever
// chose them.
#include "common.cuh"
#include "mma_utils.cuh"
#include <math.h>

namespace {
constexpr int LT = 16;                  // tokens
constexpr int L_WARPS = 16, L_THREADS = 32 * L_WARPS;
constexpr int L_CLUSTER = 8;            // CTAs that share the router's rows
constexpr int L_MAX_OUT = 512;          // router outputs
constexpr int L_MAX_PAIRS = 256;        // tokens * top
constexpr int LK = 128;                 // k of a chunk
constexpr int MOST_K = 16384;           // of a matrix of the layer (items' numbers stay within what a product divides)
constexpr float E4M3_TO_BF16 = 0x1p120f;

// An expert that some token chose: the tokens as bits, as a list (four bits each), and which of a token's choices it is (four bits a token).
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
    bf16 *h_hi, *h_lo;                  // [tokens * top + tokens, h_row]
    int h_row;
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

// 128 k of rows g and g + 8 of a warp's 16 (g = lane / 4): lane % 4 holds every fourth 16 bytes.
template <bool CODES> struct Chunk {
    static constexpr int STEPS = CODES ? 2 : 4;
    static constexpr int AHEAD = CODES ? 3 : 2;         // chunks that a warp holds or waits for
    uint4 a[STEPS][2];
    float scale[2];             // codes: of row g, of row g + 8
};
template <bool CODES>
__device__ __forceinline__ void load_chunk(Chunk<CODES>& c, const unsigned char* row0, const unsigned char* row1, int k0, int K, int lane) {
    constexpr int PER = CODES ? 16 : 8;             // k in 16 bytes
#pragma unroll
    for (int s = 0; s < Chunk<CODES>::STEPS; ++s) {
        const int k = k0 + s * 4 * PER + (lane & 3) * PER;
        const bool in = k < K;
        c.a[s][0] = in ? stream16(row0 + (long long)k * (CODES ? 1 : 2)) : make_uint4(0, 0, 0, 0);
        c.a[s][1] = in ? stream16(row1 + (long long)k * (CODES ? 1 : 2)) : make_uint4(0, 0, 0, 0);
    }
}

// Four codes as bfloat16: the even ones and the odd ones.  An e4m3's bits moved to a bfloat16's places are its value times 2^-120, subnormal ones included.
__device__ __forceinline__ void widen_codes(uint32_t w, uint32_t& even, uint32_t& odd) {
    const __nv_bfloat162 up = __float2bfloat162_rn(E4M3_TO_BF16);
    auto place = [&](uint32_t v) {
        const uint32_t bits = ((v >> 4) & 0x07f007f0u) | (v & 0x80008000u);
        const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&bits), up);
        return *reinterpret_cast<const uint32_t*>(&r);
    };
    even = place(w << 8);
    odd = place(w);
}

// d += chunk * the sum of a column's rows: `rows` are this lane's column's (lane / 4) rows of bfloat16 from the chunk's first k on, or null (a column of zeros);
// `left`: k from there on.  All of the rows are asked for before the first is used.
template <bool CODES, int ROWS>
__device__ __forceinline__ void multiply(const Chunk<CODES>& c, const bf16* const (&rows)[ROWS], int left, int lane, float (&d)[4]) {
    constexpr int PER = CODES ? 16 : 8, VECS = PER / 8, STEPS = Chunk<CODES>::STEPS;
    uint4 b[STEPS][ROWS][VECS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
#pragma unroll
            for (int v = 0; v < VECS; ++v) {
                const int k = (s * 4 + (lane & 3)) * PER + v * 8;
                b[s][i][v] = rows[i] != nullptr && k < left ? *reinterpret_cast<const uint4*>(rows[i] + k) : make_uint4(0, 0, 0, 0);
            }
    float part[4] = {};
    float(&sum)[4] = CODES ? part : d;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const uint32_t r0[4] = {c.a[s][0].x, c.a[s][0].y, c.a[s][0].z, c.a[s][0].w}, r1[4] = {c.a[s][1].x, c.a[s][1].y, c.a[s][1].z, c.a[s][1].w};
        if constexpr (CODES) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t a[4];
                widen_codes(r0[j], a[0], a[2]);
                widen_codes(r1[j], a[1], a[3]);
#pragma unroll
                for (int i = 0; i < ROWS; ++i) {
                    const uint4 v = b[s][i][j / 2];
                    const uint32_t x0 = j & 1 ? v.z : v.x, x1 = j & 1 ? v.w : v.y;
                    mma_bf16_16816(sum, a, __byte_perm(x0, x1, 0x5410), __byte_perm(x0, x1, 0x7632));
                }
            }
        } else {
            const uint32_t a0[4] = {r0[0], r1[0], r0[1], r1[1]}, a1[4] = {r0[2], r1[2], r0[3], r1[3]};
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                mma_bf16_16816(sum, a0, b[s][i][0].x, b[s][i][0].y);
                mma_bf16_16816(sum, a1, b[s][i][0].z, b[s][i][0].w);
            }
        }
    }
    if constexpr (CODES) {
        d[0] = fmaf(part[0], c.scale[0], d[0]);
        d[1] = fmaf(part[1], c.scale[0], d[1]);
        d[2] = fmaf(part[2], c.scale[1], d[2]);
        d[3] = fmaf(part[3], c.scale[1], d[3]);
    }
}

// ---- the choice ------------------------------------------------------------------------------------------------------------------------

// Bits that order floats as unsigned numbers; 0: a NaN, which is never chosen.  (-0 counts as 0.)
__device__ __forceinline__ unsigned order_of(float v) {
    if (v != v) return 0u;
    const unsigned b = __float_as_uint(v + 0.f);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logistic(float z) { return 1.0f / (1.0f + expf(-z)); }

// One warp chooses for one token: z [n_out] logits in; the scores' bits stay in the lanes (output lane + 32 i in place i).  `scratch` [n_out + n_groups] for groups.
// Lane k ends with choice k and its weight.
template <int PLACES>
__device__ __forceinline__ void choose(const LayerArgs& p, const float* z, unsigned* scratch, int lane, int& chosen, float& weight) {
    const int n = p.n_out;
    float score[PLACES];
    unsigned key[PLACES];
#pragma unroll
    for (int i = 0; i < PLACES; ++i) {
        const int e = lane + 32 * i;
        score[i] = e < n ? z[e] + (p.router_bias != nullptr ? p.router_bias[e] : 0.f) : -INFINITY;
    }
    if (p.scoring == 2) {
        float mx = -INFINITY, sum = 0.f;
#pragma unroll
        for (int i = 0; i < PLACES; ++i) mx = fmaxf(mx, score[i]);
        mx = warp_max(mx);
#pragma unroll
        for (int i = 0; i < PLACES; ++i)
            if (lane + 32 * i < n) sum += score[i] = expf(score[i] - mx);
        sum = warp_sum(sum);
#pragma unroll
        for (int i = 0; i < PLACES; ++i) score[i] = score[i] / sum;
    } else if (p.scoring == 0) {
#pragma unroll
        for (int i = 0; i < PLACES; ++i) score[i] = logistic(score[i]);
    }
#pragma unroll
    for (int i = 0; i < PLACES; ++i) {
        const int e = lane + 32 * i;
        key[i] = e < n ? order_of(score[i] + (p.correction != nullptr ? p.correction[e] : 0.f)) : 0u;
    }
    if (p.n_groups > 1) {
        // a group's rank is its best choice score; a group is kept when fewer than keep_groups rank before it (ties: the lower one first)
        const int per = n / p.n_groups;
        unsigned* best = scratch + n;
#pragma unroll
        for (int i = 0; i < PLACES; ++i)
            if (lane + 32 * i < n) scratch[lane + 32 * i] = key[i];
        __syncwarp();
        for (int g = lane; g < p.n_groups; g += 32) {
            unsigned m = 0u;
            for (int e = g * per; e < (g + 1) * per; ++e) m = max(m, scratch[e]);
            best[g] = m;
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < PLACES; ++i) {
            const int e = lane + 32 * i;
            if (e >= n) continue;
            const int g = e / per;
            int before = 0;
            for (int o = 0; o < p.n_groups; ++o) before += best[o] > best[g] || (best[o] == best[g] && o < g);
            if (before >= p.keep_groups) key[i] = 0u;
        }
    }
    chosen = 0;
    weight = 0.f;
    unsigned taken = 0u;            // this lane's places that are chosen
    for (int k = 0; k < p.top; ++k) {
        unsigned best = 0u;
        int at = 0;
#pragma unroll
        for (int i = 0; i < PLACES; ++i)
            if (key[i] > best) {
                best = key[i];
                at = i;
            }
        const unsigned m = __reduce_max_sync(0xffffffffu, best);
        unsigned e;
        if (m != 0u) {
            e = __reduce_min_sync(0xffffffffu, best == m ? (unsigned)(lane + 32 * at) : 0xffffffffu);
        } else {
            // nothing is left that compares: the first output that is not chosen yet
            const int free = __ffs((int)~taken) - 1;
            e = __reduce_min_sync(0xffffffffu, free < PLACES && lane + 32 * free < n ? (unsigned)(lane + 32 * free) : 0xffffffffu);
        }
        const int place = (int)(e >> 5);
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < PLACES; ++i)
            if (i == place) {
                s = score[i];
                if (lane == (int)(e & 31u)) {
                    key[i] = 0u;
                    taken |= 1u << i;
                }
            }
        s = __shfl_sync(0xffffffffu, s, (int)(e & 31u));
        if (lane == k) {
            chosen = (int)e;
            weight = s;
        }
    }
    const bool mine = lane < p.top;
    if (p.scoring == 1) {               // the softmax over the chosen logits
        const float mx = warp_max(mine ? weight : -INFINITY), v = mine ? expf(weight - mx) : 0.f;
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

constexpr int TEAM = 4, TEAMS = L_WARPS / TEAM;             // warps that share an item's k

struct UpShared {
    float reduce[2][L_WARPS][16][LT + 1];       // the warps' sums of 16 rows (two sets in turn); before that the router's
    LayerPlan plan;
    float gate[LT];
    unsigned long long choice[L_MAX_OUT];       // which of a token's choices an expert is, four bits a token
    unsigned tokens[L_MAX_OUT];                 // the tokens that chose an expert
};

// This CTA's rows of the router against all tokens, into every CTA's z [LT][z_row].  Sixteen rows at a time; the warps share k: a warp takes 128 k of the
// sixteen rows as three bfloat16 each.
__device__ __forceinline__ void router_logits(const LayerArgs& p, UpShared& sh, float* z, int z_row, int rank, int cluster) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2;
    const int rows = p.n_out + p.shared_gate, per = (rows + cluster - 1) / cluster, first = rank * per, mine = max(0, min(per, rows - first));
    const int tiles = (per + 15) / 16, n_chunks = (p.width + LK - 1) / LK;
    const bool second = p.n_tokens > 8;
    bool met = false;
    for (int tile = 0; tile < tiles; ++tile) {
        float acc[2][4] = {};
        const int r0 = tile * 16 + g, r1 = r0 + 8;
        const float *w0 = p.router + (long long)(first + min(r0, mine - 1)) * p.width, *w1 = p.router + (long long)(first + min(r1, mine - 1)) * p.width;
        for (int chunk = warp; chunk < n_chunks && tile * 16 < mine; chunk += L_WARPS) {
            const int k0 = chunk * LK + (lane & 3) * 8;
            float4 a[4][2][2];
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int k = k0 + s * 32;
                    a[s][0][h] = k < p.width ? *reinterpret_cast<const float4*>(w0 + k + 4 * h) : make_float4(0, 0, 0, 0);
                    a[s][1][h] = k < p.width ? *reinterpret_cast<const float4*>(w1 + k + 4 * h) : make_float4(0, 0, 0, 0);
                }
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                uint4 x[2];
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const int k = k0 + s * 32, t = n * 8 + g;
                    x[n] = k < p.width && t < p.n_tokens ? *reinterpret_cast<const uint4*>(p.x + t * p.ldx + k) : make_uint4(0, 0, 0, 0);
                }
                float v[2][8];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    v[r][0] = a[s][r][0].x, v[r][1] = a[s][r][0].y, v[r][2] = a[s][r][0].z, v[r][3] = a[s][r][0].w;
                    v[r][4] = a[s][r][1].x, v[r][5] = a[s][r][1].y, v[r][6] = a[s][r][1].z, v[r][7] = a[s][r][1].w;
                }
#pragma unroll
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
                    for (int n = 0; n < 2; ++n) {
                        if (n == 1 && !second) break;
                        mma_bf16_16816(acc[n], a0, x[n].x, x[n].y);
                        mma_bf16_16816(acc[n], a1, x[n].z, x[n].w);
                    }
                }
            }
        }
        float(*sums)[LT + 1] = sh.reduce[tile & 1][warp];
        const int col = (lane & 3) * 2;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
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
                for (int i = 0; i < L_WARPS; ++i) v += sh.reduce[tile & 1][i][r][t];
                for (int c = 0; c < cluster; ++c) st_cluster_f32(z + t * z_row + first + tile * 16 + r, v, (uint32_t)c);
            }
        }
    }
}

template <bool CODES>
__global__ __launch_bounds__(L_THREADS, 1) void moe_layer_up_kernel(const LayerArgs p) {
    extern __shared__ __align__(16) unsigned char up_smem[];
    UpShared& sh = *reinterpret_cast<UpShared*>(up_smem);
    float* z = reinterpret_cast<float*>(up_smem + sizeof(UpShared));                     // [LT][z_row]: logits, later the weights of what was chosen
    const int z_row = p.n_out + 1;
    unsigned* scratch = reinterpret_cast<unsigned*>(z + LT * z_row);                     // [L_WARPS][n_out + n_groups], with groups
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2;
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    for (int e = threadIdx.x; e < p.n_out; e += L_THREADS) {
        sh.tokens[e] = 0u;
        sh.choice[e] = 0ull;
    }
    pdl_wait();
    router_logits(p, sh, z, z_row, blockIdx.x % L_CLUSTER, L_CLUSTER);
    cluster_sync_all();

    if (warp < p.n_tokens) {
        int e;
        float w;
        unsigned* mine = scratch + warp * (p.n_out + p.n_groups);
        if (p.n_out <= 128) choose<4>(p, z + warp * z_row, mine, lane, e, w);
        else choose<L_MAX_OUT / 32>(p, z + warp * z_row, mine, lane, e, w);
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
    int n_active = 0;
    for (int c = 0; c * 32 < p.n_real; ++c) {
        const int e = c * 32 + lane;
        const unsigned tokens = e < p.n_real ? sh.tokens[e] : 0u, votes = __ballot_sync(0xffffffffu, tokens != 0u);
        if (warp == c % L_WARPS && tokens != 0u) {
            ActiveExpert& a = sh.plan.of[n_active + __popc(votes & ((1u << lane) - 1u))];
            unsigned long long list = 0ull;
            int n = 0;
            for (unsigned m = tokens; m != 0u; m &= m - 1u, ++n) list |= (unsigned long long)(__ffs((int)m) - 1) << (4 * n);
            a.expert = e;
            a.tokens = tokens;
            a.list = list;
            a.choice = sh.choice[e];
        }
        n_active += __popc(votes);
    }
    if (threadIdx.x == 0) sh.plan.n_active = n_active;
    __syncthreads();
    if (blockIdx.x == 0) {
        const int words = (int)(offsetof(LayerPlan, of) + (size_t)n_active * sizeof(ActiveExpert)) / 8;
        for (int i = threadIdx.x; i < words; i += L_THREADS) reinterpret_cast<unsigned long long*>(p.plan)[i] = reinterpret_cast<const unsigned long long*>(&sh.plan)[i];
    }
    pdl_trigger();

    // items: eight features of the shared expert, then of every active one; a team's warp takes every TEAM-th chunk of their k, a round each
    const int shared_items = p.inner_shared / 8, per_expert = p.inner / 8, n_items = shared_items + n_active * per_expert;
    const int n_chunks = (p.width + LK - 1) / LK, rounds = (n_chunks + TEAM - 1) / TEAM;
    const int team = warp / TEAM, member = warp % TEAM, stride = gridDim.x * TEAMS, first = team * gridDim.x + blockIdx.x;
    auto active_of = [&](int item) { return quotient(item - shared_items, p.per_expert_magic); };
    auto load = [&](Chunk<CODES>& c, int item, int round) {
        if (item >= n_items) return;
        const bool own = item >= shared_items;
        const int a = own ? active_of(item) : 0, f = (own ? item - shared_items - a * per_expert : item) * 8 + g, e = own ? sh.plan.of[a].expert : 0;
        const LayerMatrix& m = own ? p.up : p.shared_up;
        const int il = own ? p.interleave : p.interleave_shared, chunk = member + round * TEAM;
        // row g of the 16 is a gate row, row g + 8 the row of the linear branch of the same feature
        const int r0 = il == 0 ? f : il == 4 ? 2 * f - (f & 3) : f / il * 2 * il + f % il, r1 = r0 + (il > 0 ? il : own ? p.inner : p.inner_shared);
        const unsigned char* base = m.w + e * m.stack_bytes;
        load_chunk<CODES>(c, base + r0 * m.row_bytes, base + r1 * m.row_bytes, chunk * LK, p.width, lane);
        if (CODES) {
            const float* scales = m.scales + (long long)e * m.row_blocks * m.k_blocks + min(chunk, n_chunks - 1);
            c.scale[0] = scales[(long long)(r0 / LK) * m.k_blocks];
            c.scale[1] = scales[(long long)(r1 / LK) * m.k_blocks];
        }
    };
    constexpr int AHEAD = Chunk<CODES>::AHEAD;
    Chunk<CODES> held[AHEAD];
    int to_load = first, load_round = 0;
    auto load_next = [&](Chunk<CODES>& c) {
        load(c, to_load, load_round);
        if (++load_round == rounds) {
            load_round = 0;
            to_load += stride;
        }
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) load_next(held[i]);
    float acc[2][4];
    const bf16 *row0 = nullptr, *row1 = nullptr;
    int n_cols = 0, set = 0;
    for (int item = first, round = 0; item < n_items;) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (item >= n_items) break;
            const bool own = item >= shared_items;
            const int a = own ? active_of(item) : 0;
            if (round == 0) {
                // this lane's columns: the tokens that chose the expert, or all for the shared one
                const unsigned long long list = own ? sh.plan.of[a].list : 0xfedcba9876543210ull;
                n_cols = own ? __popc(sh.plan.of[a].tokens) : p.n_tokens;
                row0 = g < n_cols ? p.x + (long long)((list >> (4 * g)) & 15) * p.ldx : nullptr;
                row1 = 8 + g < n_cols ? p.x + (long long)((list >> (32 + 4 * g)) & 15) * p.ldx : nullptr;
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[n][j] = 0.f;
            }
            const int chunk = member + round * TEAM, k0 = chunk * LK;
            if (chunk < n_chunks) {
                const bf16* at[1] = {row0 != nullptr ? row0 + k0 : nullptr};
                multiply<CODES, 1>(held[i], at, p.width - k0, lane, acc[0]);
                if (n_cols > 8) {
                    const bf16* at1[1] = {row1 != nullptr ? row1 + k0 : nullptr};
                    multiply<CODES, 1>(held[i], at1, p.width - k0, lane, acc[1]);
                }
            }
            load_next(held[i]);
            if (++round < rounds) continue;
            const int f0 = (own ? item - shared_items - a * per_expert : item) * 8;
            round = 0;
            item += stride;
            float(*mine)[LT + 1] = sh.reduce[set][warp];
            const int col = (lane & 3) * 2;
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                if (n == 1 && n_cols <= 8) break;
                mine[g][n * 8 + col] = acc[n][0];
                mine[g][n * 8 + col + 1] = acc[n][1];
                mine[g + 8][n * 8 + col] = acc[n][2];
                mine[g + 8][n * 8 + col + 1] = acc[n][3];
            }
            // (two sets in turn: nobody writes this one again before the team has come to the next item's barrier)
            asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(32 * TEAM) : "memory");
            const int f = lane & 7, c = member * 4 + (lane >> 3);
            if (c < n_cols) {
                float gate = 0.f, lin = 0.f;
#pragma unroll
                for (int w = 0; w < TEAM; ++w) {
                    gate += sh.reduce[set][team * TEAM + w][f][c];
                    lin += sh.reduce[set][team * TEAM + w][f + 8][c];
                }
                if (p.limit != INFINITY) {          // (a NaN stays one)
                    gate = gate > p.limit ? p.limit : gate;
                    lin = lin > p.limit ? p.limit : lin < -p.limit ? -p.limit : lin;
                }
                int row, t = c;
                float w;
                if (own) {
                    const ActiveExpert& ex = sh.plan.of[a];
                    t = (int)(ex.list >> (4 * c)) & 15;
                    row = t * p.top + ((int)(ex.choice >> (4 * t)) & 15);
                    w = z[t * z_row + ex.expert];
                } else {
                    row = p.n_tokens * p.top + t;
                    w = sh.gate[t];
                }
                const float v = glu_gate(gate, p.slope) * (lin + p.shift) * w;
                const bf16 hi = __float2bfloat16_rn(v);
                const long long at = (long long)row * p.h_row + f0 + f;
                p.h_hi[at] = hi;
                p.h_lo[at] = __float2bfloat16_rn(v - __bfloat162float(hi));
            }
            set ^= 1;
        }
    }
}

// ---- down ------------------------------------------------------------------------------------------------------------------------------

struct DownShared {
    float reduce[L_WARPS][16][LT + 1];
    float cluster[16][LT];
    LayerPlan plan;
};

// CTA r of a cluster of `parts` takes its share of the chunks of 16 output features; a cluster takes features 16 (blockIdx / parts), ...
template <bool CODES>
__global__ __launch_bounds__(L_THREADS, 1) void moe_layer_down_kernel(const LayerArgs p, int parts) {
    extern __shared__ __align__(16) unsigned char down_smem[];
    DownShared& sh = *reinterpret_cast<DownShared*>(down_smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2;
    const int rank = blockIdx.x % parts, clusters = gridDim.x / parts, n_groups = (p.width + 15) / 16;
    pdl_wait();
    // (as much of the plan as the step can have: its length comes with it)
    const int words = (int)(offsetof(LayerPlan, of) + (size_t)min(p.n_tokens * p.top, p.n_real) * sizeof(ActiveExpert)) / 8;
    for (int i = threadIdx.x; i < words; i += L_THREADS) reinterpret_cast<unsigned long long*>(&sh.plan)[i] = reinterpret_cast<const unsigned long long*>(p.plan)[i];
    __syncthreads();
    pdl_trigger();
    const int own_chunks = (p.inner + LK - 1) / LK, shared_chunks = (p.inner_shared + LK - 1) / LK, n_chunks = shared_chunks + sh.plan.n_active * own_chunks;
    auto active_of = [&](int chunk) { return quotient(chunk - shared_chunks, p.own_chunks_magic); };
    const int step = parts * L_WARPS, first = rank * L_WARPS + warp;
    auto load = [&](Chunk<CODES>& c, int group, int chunk) {
        const bool own = chunk >= shared_chunks;
        const int a = own ? active_of(chunk) : 0, kb = own ? (chunk - shared_chunks) - a * own_chunks : chunk;
        const bool some = chunk < n_chunks;
        const int e = own && some ? sh.plan.of[a].expert : 0;
        const LayerMatrix& m = own ? p.down : p.shared_down;
        const int r0 = min(group * 16 + g, p.width - 1), r1 = min(group * 16 + g + 8, p.width - 1);
        const unsigned char* base = m.w + e * m.stack_bytes;
        load_chunk<CODES>(c, base + r0 * m.row_bytes, base + r1 * m.row_bytes, kb * LK, some ? own ? p.inner : p.inner_shared : 0, lane);
        if (CODES && some) {
            const float* s = m.scales + (long long)e * m.row_blocks * m.k_blocks;
            c.scale[0] = s[(long long)(r0 / LK) * m.k_blocks + kb];
            c.scale[1] = s[(long long)(r1 / LK) * m.k_blocks + kb];
        }
    };
    float acc[2][4];
    auto work = [&](const Chunk<CODES>& c, int chunk) {
        if (chunk >= n_chunks) return;
        const bool own = chunk >= shared_chunks;
        const int a = own ? active_of(chunk) : 0, kb = own ? (chunk - shared_chunks) - a * own_chunks : chunk;
        const unsigned tokens = own ? sh.plan.of[a].tokens : (1u << p.n_tokens) - 1u;
        const unsigned long long choice = own ? sh.plan.of[a].choice : 0ull;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            if ((tokens >> (8 * n) & 0xffu) == 0u) continue;                // (none of these eight columns)
            const int t = n * 8 + g, row = own ? t * p.top + ((int)(choice >> (4 * t)) & 15) : p.n_tokens * p.top + t;
            const long long at = (long long)row * p.h_row + kb * LK;
            const bool have = tokens >> t & 1u;
            const bf16* rows[2] = {have ? p.h_hi + at : nullptr, have ? p.h_lo + at : nullptr};
            multiply<CODES, 2>(c, rows, (own ? p.inner : p.inner_shared) - kb * LK, lane, acc[n]);
        }
    };
    constexpr int AHEAD = Chunk<CODES>::AHEAD;
    const int rounds = max(1, (n_chunks + step - 1) / step), turns = (rounds + AHEAD - 1) / AHEAD * AHEAD;       // (empty chunks fill the last turn)
    Chunk<CODES> held[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) load(held[i], blockIdx.x / parts, first + i * step);
    for (int group = blockIdx.x / parts; group < n_groups; group += clusters) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
        for (int round = 0; round < turns; round += AHEAD) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                work(held[i], first + (round + i) * step);
                if (round + AHEAD < turns) load(held[i], group, first + (round + i + AHEAD) * step);
                else if (group + clusters < n_groups) load(held[i], group + clusters, first + i * step);
            }
        }
        const int col = (lane & 3) * 2;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            sh.reduce[warp][g][n * 8 + col] = acc[n][0];
            sh.reduce[warp][g][n * 8 + col + 1] = acc[n][1];
            sh.reduce[warp][g + 8][n * 8 + col] = acc[n][2];
            sh.reduce[warp][g + 8][n * 8 + col + 1] = acc[n][3];
        }
        __syncthreads();
        const int f = threadIdx.x & 15, t = threadIdx.x >> 4;
        float v = 0.f;
        if (t < p.n_tokens) {
#pragma unroll
            for (int i = 0; i < L_WARPS; ++i) v += sh.reduce[i][f][t];
            if (parts > 1) sh.cluster[f][t] = v;
        }
        if (parts > 1) {
            cluster_sync_all();
            if (rank == 0 && t < p.n_tokens)
                for (int r = 1; r < parts; ++r) v += ld_dsmem(&sh.cluster[f][t], (uint32_t)r);
            cluster_sync_all();
        } else {
            __syncthreads();
        }
        const int feature = group * 16 + f;
        if (rank == 0 && t < p.n_tokens && feature < p.width) {
            const float w = sh.plan.identity[t];
            if (p.n_out > p.n_real) v += w * __bfloat162float(p.x[(long long)t * p.ldx + feature]);
            p.out[(long long)t * p.width + feature] = __float2bfloat16_rn(v);
        }
    }
}

size_t up_smem_bytes(const LayerArgs& p) {
    return sizeof(UpShared) + (size_t)LT * (p.n_out + 1) * 4 + (p.n_groups > 1 ? (size_t)L_WARPS * (p.n_out + p.n_groups) * 4 : 0);
}

// Clusters of the up kernel that the device holds at once (asked for once a device): a grid that needs a second round would route twice.
template <bool CODES> int up_clusters(size_t smem) {
    static std::atomic<int> known[64];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 1;
    if (dev < 64 && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(64 * L_CLUSTER);
    cfg.blockDim = dim3(L_THREADS);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = L_CLUSTER;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, moe_layer_up_kernel<CODES>, &cfg) != cudaSuccess || n < 1) n = 1;
    if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
    return n;
}

template <bool CODES> int launch_layer(const LayerArgs& p, int sms, cudaStream_t stream) {
    static std::atomic<unsigned long long> allowed_up{0}, allowed_down{0};
    cudaError_t e = rlis_allow_smem(moe_layer_up_kernel<CODES>, 200 * 1024, allowed_up);
    if (e == cudaSuccess) e = rlis_allow_smem(moe_layer_down_kernel<CODES>, (int)sizeof(DownShared), allowed_down);
    if (e != cudaSuccess) return (int)e;
    const int clusters = up_clusters<CODES>(up_smem_bytes(p));
    rlis_launch_cluster(moe_layer_up_kernel<CODES>, dim3((unsigned)(clusters * L_CLUSTER)), dim3(L_THREADS), up_smem_bytes(p), stream, dim3(L_CLUSTER, 1, 1), p);
    const int rc = RLIS_LAUNCH_CHECK();
    if (rc != 0) return rc;
    const int groups = (p.width + 15) / 16;
    int parts = 1;
    while (parts < 4 && groups * parts * 4 < 3 * sms) parts *= 2;
    const int at_once = sms / parts < groups ? sms / parts : groups;
    rlis_launch_cluster(moe_layer_down_kernel<CODES>, dim3((unsigned)(at_once * parts)), dim3(L_THREADS), sizeof(DownShared), stream, dim3((unsigned)parts, 1, 1), p, parts);
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

// Bytes of workspace of a call.
extern "C" int rlis_moe_layer_bytes(int n_tokens, int top, int inner, int inner_shared) {
    const long long row = ((inner > inner_shared ? inner : inner_shared) + 7) / 8 * 8;
    return (int)((sizeof(LayerPlan) + 15) / 16 * 16 + 4 * (long long)(n_tokens * top + n_tokens) * row);
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
    // codes: the eight rows that a load instruction takes lie in one block of rows
    if (codes && ((a->interleave > 0 && a->interleave != 4 && a->interleave % 8 != 0) || (a->interleave_shared > 0 && a->interleave_shared != 4 && a->interleave_shared % 8 != 0)))
        return RLIS_ERR_UNSUPPORTED;
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
    p.h_row = ((a->inner > a->inner_shared ? a->inner : a->inner_shared) + 7) / 8 * 8;
    p.h_hi = reinterpret_cast<bf16*>(static_cast<unsigned char*>(a->workspace) + (sizeof(LayerPlan) + 15) / 16 * 16);
    p.h_lo = p.h_hi + (long long)(a->n_tokens * a->top + a->n_tokens) * p.h_row;
    p.out = static_cast<bf16*>(a->out);
    auto magic = [](int d) { return d > 1 ? (unsigned)(((1ull << 32) + d - 1) / d) : 0u; };
    p.per_expert_magic = magic(a->inner / 8);
    p.own_chunks_magic = magic((a->inner + LK - 1) / LK);
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (up_smem_bytes(p) > 200 * 1024) return RLIS_ERR_UNSUPPORTED;
    return codes ? launch_layer<true>(p, sms, stream) : launch_layer<false>(p, sms, stream);
}
