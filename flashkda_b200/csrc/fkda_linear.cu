// Linear attention with a decay for each head:
//     S_t = exp(g_t) S_{t-1} + v_t k_t^T  ([V, K]),   o_t = scale S_t q_t
//
// Prompts go through chunks of 64 tokens.  With G the running sum of g in a chunk and S the state in front of it,
//     O = scale (P V + diag(exp(G)) Q S^T),   P_ij = exp(G_i - G_j) (q_i . k_j) for j <= i
//     S' = exp(G_64) S + (diag(w) V)^T K,     w_j = exp(G_64 - G_j)
// All four products run on tcgen05: q k^T and the two of O as accumulators of 64 rows, the state as one of 128 x 128 that stays in
// tensor memory for the whole sequence.  The call is bound by HBM (1 KB per token and head against 2 x 128 x (64 + 128 + 128)
// operations), so one CTA walks a (sequence, head) chain with everything between the copies in and out on the chip, and a chunk's
// stages are spread over warpgroups: state (read, rounded for Q S^T, decayed, written back), scores and outputs, weighted
// values, one warp each for the copies, the products and the decays.
//
// Numerics: decays are sums of g in fp32 over at most 64 tokens, w as sums over the tokens behind j (no differences of large sums).
// P and the copy of S that Q multiplies are rounded to bf16, which the bf16 outputs do not show.  The state is not rounded: it
// is fp32 throughout, and w V enters the product as three bf16 terms, which hold all 24 bits.
//
// Single tokens: a read-modify-write of the state by a kernel of its own, as bound by HBM as that is.
#include "fkda_tc5.cuh"

namespace fkda {
namespace {

using namespace tc5;

constexpr int kC = 64;                        // tokens of a chunk
constexpr int kTileBytes = kC * 128;          // 64 tokens x 64 dimensions
constexpr int kOperandBytes = 2 * kTileBytes; // a chunk of q, k or v
constexpr int kStageBytes = 3 * kOperandBytes;
constexpr int kStages = 2;
constexpr int kTerms = 3;
constexpr int kThreads = 480;
constexpr int kOffSplit = kStages * kStageBytes;
constexpr int kOffState = kOffSplit + kTerms * kOperandBytes;
constexpr int kOffOut = kOffState + kD * kD * 2;
constexpr int kOffBars = kOffOut + kC * kD * 2;
constexpr uint32_t kS = 0, kScore = 128, kO1 = 256, kO2 = 384;   // tensor-memory columns

struct LinearArgs {
    const float* g;
    __nv_bfloat16 *q, *k, *v, *out;
    const void* h0;
    void* hT;
    const int64_t* cu;
    int64_t T, N, g_batch, g_token, g_head, out_batch, out_token, out_head;
    int64_t q_batch, q_token, q_head, k_batch, k_token, k_head, v_batch, v_token, v_head;
    int H, group;      // value heads, value heads of a key head
    float scale;
    bool state_fp32, skip_single;
};
struct LinearMaps {
    CUtensorMap q, k, v;
};
struct Decays {
    float G[kC], eG[kC], w[kC], total;
    float pad[3];
};
struct Bars {
    Decays decay[2];
    uint64_t full[kStages], empty[kStages], dec_full[2], dec_empty[2], score[2], p_full, out_full, out_free, s_ready, s_done, split_full, drained;
    uint32_t tmem;
    int abort;
};
constexpr int kSmem = 1024 + kOffBars + ((int)sizeof(Bars) + 127) / 128 * 128;
static_assert(kSmem <= 232448, "shared memory of an SM");

constexpr float kLog2e = 1.4426950408889634f;
// exp(-100) is nothing in fp32; a decay below it (minus infinity to start afresh) would make differences of sums meaningless.
__device__ __forceinline__ float log2_decay(float g) { return (g < -100.0f ? -100.0f : g) * kLog2e; }

struct Chain {
    int64_t n, b, t0;
    int h, len;
};
__device__ __forceinline__ Chain locate(const LinearArgs& a, int64_t chain) {
    Chain c;
    c.n = chain / a.H;
    c.h = (int)(chain - c.n * a.H);
    if (a.cu == nullptr) {
        c.b = c.n;
        c.t0 = 0;
        c.len = (int)a.T;
    } else {
        c.b = 0;
        const int64_t lo = a.cu[c.n] < 0 ? 0 : a.cu[c.n], hi = a.cu[c.n + 1] > a.T ? a.T : a.cu[c.n + 1];
        c.t0 = lo;
        c.len = hi > lo ? (int)(hi - lo) : 0;
    }
    return c;
}

// 32 numbers of a row of the state
__device__ __forceinline__ void load_state32(const LinearArgs& a, int64_t at, uint32_t* r) {
    if (a.h0 == nullptr) {
#pragma unroll
        for (int i = 0; i < 32; ++i) r[i] = 0u;
    } else if (a.state_fp32) {
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const float*>(a.h0) + at);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint4 x = src[i];
            r[4 * i] = x.x; r[4 * i + 1] = x.y; r[4 * i + 2] = x.z; r[4 * i + 3] = x.w;
        }
    } else {
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.h0) + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 x = src[i];
            const uint32_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                r[8 * i + 2 * j] = y[j] << 16;
                r[8 * i + 2 * j + 1] = y[j] & 0xffff0000u;
            }
        }
    }
}
__device__ __forceinline__ void store_state32(const LinearArgs& a, int64_t at, const uint32_t* r) {
    if (a.state_fp32) {
        uint4* dst = reinterpret_cast<uint4*>(static_cast<float*>(a.hT) + at);
#pragma unroll
        for (int i = 0; i < 8; ++i) dst[i] = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
    } else {
        uint4* dst = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.hT) + at);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            dst[i] = make_uint4(pack_bf2(f(r[8 * i]), f(r[8 * i + 1])), pack_bf2(f(r[8 * i + 2]), f(r[8 * i + 3])),
                                pack_bf2(f(r[8 * i + 4]), f(r[8 * i + 5])), pack_bf2(f(r[8 * i + 6]), f(r[8 * i + 7])));
    }
}

__global__ void __launch_bounds__(kThreads, 1) linear_chunk_kernel(const __grid_constant__ LinearArgs a, const __grid_constant__ LinearMaps maps) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    Bars& bar = *reinterpret_cast<Bars*>(smem + kOffBars);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) mbar_init(&bar.full[i], 1), mbar_init(&bar.empty[i], 1);
        for (int i = 0; i < 2; ++i) mbar_init(&bar.dec_full[i], 1), mbar_init(&bar.dec_empty[i], 12), mbar_init(&bar.score[i], 1);
        mbar_init(&bar.p_full, 128);
        mbar_init(&bar.out_full, 1);
        mbar_init(&bar.out_free, 128);
        mbar_init(&bar.s_ready, 128);
        mbar_init(&bar.s_done, 1);
        mbar_init(&bar.split_full, 128);
        mbar_init(&bar.drained, 1);
        bar.abort = 0;
        mbar_fence_init();
    }
    if (warp == 13) tmem_alloc(&bar.tmem, 512);
    fence_before();
    grid_dep_launch();
    grid_dep_wait();
    __syncthreads();
    fence_after();
    const uint32_t tmem = bar.tmem;
    const Chain ch = locate(a, blockIdx.x);
    const bool mine = !(a.skip_single && ch.len <= 1);
    const int n = mine ? (ch.len + kC - 1) / kC : 0;

    if (warp == 12) {
        // ---- copies ----
        if (elect_one()) {
            bool ok = true;
            int c = 0;
            for (; c < n; ++c) {
                const int s = c % kStages;
                if (c >= kStages) ok = wait(&bar.empty[s], (c / kStages - 1) & 1, &bar.abort);
                if (!ok) break;
                uint8_t* dst = smem + s * kStageBytes;
                const int t = (int)ch.t0 + c * kC;
                mbar_arrive_expect_tx(&bar.full[s], kStageBytes);
                for (int x = 0; x < 2; ++x) {
                    tma_load_4d(dst + x * kTileBytes, &maps.q, x * 64, ch.h / a.group, t, (int)ch.b, &bar.full[s]);
                    tma_load_4d(dst + kOperandBytes + x * kTileBytes, &maps.k, x * 64, ch.h / a.group, t, (int)ch.b, &bar.full[s]);
                    tma_load_4d(dst + 2 * kOperandBytes + x * kTileBytes, &maps.v, x * 64, ch.h, t, (int)ch.b, &bar.full[s]);
                }
            }
            for (int k = max(0, c - kStages); k < c; ++k) drain(&bar.full[k % kStages], (k / kStages) & 1);
        }
    } else if (warp == 13) {
        // ---- products ----
        if (n > 0 && elect_one()) {
            const uint32_t base = smem_u32(smem), split = base + kOffSplit, state = base + kOffState;
            constexpr uint32_t kIdScore = idesc(64, 64, false, false), kIdOut1 = idesc(64, 128, false, false),
                               kIdOut2 = idesc(64, 128, false, true), kIdState = idesc(128, 128, true, true);
            bool ok = true;
            auto score = [&](int c) {
                ok = wait(&bar.full[c % kStages], (c / kStages) & 1, &bar.abort);
                if (!ok) return;
                fence_after();
                const uint32_t q = base + (c % kStages) * kStageBytes, k = q + kOperandBytes;
                for (int x = 0; x < 2; ++x)
                    for (int i = 0; i < 4; ++i)
                        mma_ss(tmem + kScore + (c & 1) * 64, desc(q + x * kTileBytes + i * 32), desc(k + x * kTileBytes + i * 32), kIdScore, (x | i) != 0);
                commit(&bar.score[c & 1]);   // (one barrier per buffer: chunk c + 1's scores may be there before chunk c's outputs are away)
            };
            score(0);
            for (int c = 0; c < n && ok; ++c) {
                const uint32_t q = base + (c % kStages) * kStageBytes, k = q + kOperandBytes, v = k + kOperandBytes;
                ok = wait(&bar.s_ready, c & 1, &bar.abort) && (c == 0 || wait(&bar.out_free, (c - 1) & 1, &bar.abort));
                if (!ok) break;
                fence_after();
                for (int x = 0; x < 2; ++x)
                    for (int i = 0; i < 4; ++i)
                        mma_ss(tmem + kO1, desc(q + x * kTileBytes + i * 32), desc(state + x * (kD * 128) + i * 32), kIdOut1, (x | i) != 0);
                ok = wait(&bar.split_full, c & 1, &bar.abort);
                if (!ok) break;
                fence_after();
                for (int t = 0; t < kTerms; ++t)
                    for (int i = 0; i < 4; ++i)
                        mma_ss(tmem + kS, desc(split + t * kOperandBytes + i * 2048, kTileBytes), desc(k + i * 2048, kTileBytes), kIdState, 1);
                commit(&bar.s_done);
                if (c + 1 < n) score(c + 1);
                if (!ok) break;
                ok = wait(&bar.p_full, c & 1, &bar.abort);
                if (!ok) break;
                fence_after();
                for (int i = 0; i < 4; ++i)
                    mma_ts(tmem + kO2, tmem + kScore + (c & 1) * 64 + i * 8, desc(v + i * 2048, kTileBytes), kIdOut2, i != 0);
                commit(&bar.out_full);
                commit(&bar.empty[c % kStages]);
            }
            commit(&bar.drained);
            drain(&bar.drained, 0);
        }
    } else if (warp == 14) {
        // ---- decays: lane l has tokens 2 l and 2 l + 1 of a chunk ----
        const float* g = a.g + ch.b * a.g_batch + ch.t0 * a.g_token + ch.h * a.g_head;
        for (int c = 0; c < n; ++c) {
            const int t = c * kC + 2 * lane;
            const float x = t < ch.len ? log2_decay(g[t * a.g_token]) : 0.0f, y = t + 1 < ch.len ? log2_decay(g[(t + 1) * a.g_token]) : 0.0f;
            float upto = x + y, from = x + y;   // sums over the lanes up to mine, and from mine on
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const float p = __shfl_up_sync(0xffffffffu, upto, off), q = __shfl_down_sync(0xffffffffu, from, off);
                if (lane >= off) upto += p;
                if (lane + off < 32) from += q;
            }
            const float before = __shfl_up_sync(0xffffffffu, upto, 1), behind = __shfl_down_sync(0xffffffffu, from, 1);
            const float G0 = (lane > 0 ? before : 0.0f) + x, G1 = G0 + y, w1 = lane < 31 ? behind : 0.0f, w0 = w1 + y;
            if (c >= 2) wait(&bar.dec_empty[c & 1], (c / 2 - 1) & 1, &bar.abort);
            Decays& d = bar.decay[c & 1];
            d.G[2 * lane] = G0;
            d.G[2 * lane + 1] = G1;
            d.eG[2 * lane] = ex2_approx(G0);
            d.eG[2 * lane + 1] = ex2_approx(G1);
            d.w[2 * lane] = ex2_approx(w0);
            d.w[2 * lane + 1] = ex2_approx(w1);
            if (lane == 0) d.total = ex2_approx(from);
            __syncwarp();
            if (lane == 0) arrive(&bar.dec_full[c & 1]);
        }
    } else if (warp < 4) {
        // ---- state: thread = row ----
        const int v = warp * 32 + lane;
        const uint32_t ts = tmem + kS + ((uint32_t)(warp * 32) << 16);
        const int64_t at = ((ch.n * a.H + ch.h) * kD + v) * (int64_t)kD;
        uint8_t* row = smem + kOffState + v * 128;
        for (int c = 0; c < n; ++c) {
            wait(&bar.dec_full[c & 1], (c >> 1) & 1, &bar.abort);
            const float total = bar.decay[c & 1].total;
            __syncwarp();
            mbar_arrive_lane0(&bar.dec_empty[c & 1], lane);
            if (c > 0) {
                wait(&bar.s_done, (c - 1) & 1, &bar.abort);
                fence_after();
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                uint32_t r[32];
                if (c > 0) {
                    ld32(ts + x * 32, r);
                    wait_ld();
                } else {
                    load_state32(a, at + x * 32, r);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<uint4*>(row + (x >> 1) * (kD * 128) + ((((x & 1) * 4 + i) ^ (v & 7)) << 4)) =
                        make_uint4(pack_bf2(f(r[8 * i]), f(r[8 * i + 1])), pack_bf2(f(r[8 * i + 2]), f(r[8 * i + 3])),
                                   pack_bf2(f(r[8 * i + 4]), f(r[8 * i + 5])), pack_bf2(f(r[8 * i + 6]), f(r[8 * i + 7])));
#pragma unroll
                for (int i = 0; i < 32; ++i) r[i] = u(f(r[i]) * total);
                st32(ts + x * 32, r);
            }
            wait_st();
            fence_proxy_async_smem();
            fence_before();
            arrive(&bar.s_ready);
        }
        if (n > 0) {
            wait(&bar.s_done, (n - 1) & 1, &bar.abort);
            fence_after();
        }
        if (mine && a.hT != nullptr) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                uint32_t r[32];
                if (n > 0) {
                    ld32(ts + x * 32, r);
                    wait_ld();
                } else {
                    load_state32(a, at + x * 32, r);
                }
                store_state32(a, at + x * 32, r);
            }
        }
        fence_before();
    } else if (warp < 8) {
        // ---- scores to weights, outputs: warp w has rows 16 w .. 16 w + 15, thread 4 g + t rows g and g + 8 of these ----
        const int w = warp - 4, gr = lane >> 2, tc = lane & 3;
        const int r0 = w * 16 + gr, r1 = r0 + 8;
        const uint32_t lanes = (uint32_t)(w * 32) << 16;
        uint8_t* stage = smem + kOffOut + w * 16 * 256;
        __nv_bfloat16* out = a.out + ch.b * a.out_batch + ch.t0 * a.out_token + ch.h * a.out_head;
        for (int c = 0; c < n; ++c) {
            wait(&bar.dec_full[c & 1], (c >> 1) & 1, &bar.abort);
            const Decays& d = bar.decay[c & 1];
            const float G0 = d.G[r0], G1 = d.G[r1], e0 = d.eG[r0] * a.scale, e1 = d.eG[r1] * a.scale;
            wait(&bar.score[c & 1], (c >> 1) & 1, &bar.abort);
            fence_after();
            uint32_t s[32], p[16];
            ld_frag64(tmem + kScore + (c & 1) * 64 + lanes, s);
            wait_ld();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (i <= 2 * w + 1) {   // (columns behind the warp's last row are masked for all of its rows)
                    const int j = 8 * i + 2 * tc;
                    const float2 G = *reinterpret_cast<const float2*>(&d.G[j]);
                    const float a0 = j <= r0 ? f(s[4 * i]) * ex2_approx(G0 - G.x) : 0.0f, a1 = j + 1 <= r0 ? f(s[4 * i + 1]) * ex2_approx(G0 - G.y) : 0.0f;
                    const float b0 = j <= r1 ? f(s[4 * i + 2]) * ex2_approx(G1 - G.x) : 0.0f, b1 = j + 1 <= r1 ? f(s[4 * i + 3]) * ex2_approx(G1 - G.y) : 0.0f;
                    p[2 * i] = pack_bf2(a0, a1);
                    p[2 * i + 1] = pack_bf2(b0, b1);
                } else {
                    p[2 * i] = p[2 * i + 1] = 0u;
                }
            }
            st_frag32(tmem + kScore + (c & 1) * 64 + lanes, p);
            wait_st();
            fence_before();
            arrive(&bar.p_full);
            __syncwarp();
            mbar_arrive_lane0(&bar.dec_empty[c & 1], lane);

            wait(&bar.out_full, c & 1, &bar.abort);
            fence_after();
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                uint32_t o1[32], o2[32];
                ld_frag64(tmem + kO1 + x * 64 + lanes, o1);
                ld_frag64(tmem + kO2 + x * 64 + lanes, o2);
                wait_ld();
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int unit = (x * 8 + i) ^ gr;
                    *reinterpret_cast<uint32_t*>(stage + gr * 256 + unit * 16 + tc * 4) =
                        pack_bf2(__fmaf_rn(f(o1[4 * i]), e0, f(o2[4 * i]) * a.scale), __fmaf_rn(f(o1[4 * i + 1]), e0, f(o2[4 * i + 1]) * a.scale));
                    *reinterpret_cast<uint32_t*>(stage + (gr + 8) * 256 + unit * 16 + tc * 4) =
                        pack_bf2(__fmaf_rn(f(o1[4 * i + 2]), e1, f(o2[4 * i + 2]) * a.scale), __fmaf_rn(f(o1[4 * i + 3]), e1, f(o2[4 * i + 3]) * a.scale));
                }
            }
            fence_before();
            arrive(&bar.out_free);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int r = 2 * i + (lane >> 4), t = c * kC + w * 16 + r;
                const uint4 x = *reinterpret_cast<const uint4*>(stage + r * 256 + (((lane & 15) ^ (r & 7)) << 4));
                if (t < ch.len) *reinterpret_cast<uint4*>(out + t * a.out_token + (lane & 15) * 8) = x;
            }
            __syncwarp();
        }
    } else {
        // ---- weighted values in three terms; rows behind the sequence's end become nothing ----
        const int me = (warp - 8) * 32 + lane;
        for (int c = 0; c < n; ++c) {
            const int s = c % kStages, valid = min(kC, ch.len - c * kC);
            uint8_t* k = smem + s * kStageBytes + kOperandBytes;
            uint8_t* v = k + kOperandBytes;
            uint8_t* split = smem + kOffSplit;
            wait(&bar.dec_full[c & 1], (c >> 1) & 1, &bar.abort);
            float w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = bar.decay[c & 1].w[i * 16 + (me >> 3)];
            __syncwarp();
            mbar_arrive_lane0(&bar.dec_empty[c & 1], lane);
            wait(&bar.full[s], (c / kStages) & 1, &bar.abort);
            if (c > 0) wait(&bar.s_done, (c - 1) & 1, &bar.abort);   // (the last chunk's terms have been read)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int at = (i * 128 + me) * 16, t = (i & 3) * 16 + (me >> 3);   // 16 bytes of token t
                uint4 x = *reinterpret_cast<const uint4*>(v + at);
                if (t >= valid) {
                    x = make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4*>(v + at) = x;
                    *reinterpret_cast<uint4*>(k + at) = x;
                }
                uint32_t in[4] = {x.x, x.y, x.z, x.w}, term[kTerms][4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float lo = bf_lo(in[j]) * w[i & 3], hi = bf_hi(in[j]) * w[i & 3];
#pragma unroll
                    for (int m = 0; m < kTerms; ++m) {
                        term[m][j] = pack_bf2(lo, hi);
                        lo -= bf_lo(term[m][j]);
                        hi -= bf_hi(term[m][j]);
                    }
                }
#pragma unroll
                for (int m = 0; m < kTerms; ++m) *reinterpret_cast<uint4*>(split + m * kOperandBytes + at) = make_uint4(term[m][0], term[m][1], term[m][2], term[m][3]);
            }
            fence_proxy_async_smem();
            arrive(&bar.split_full);
        }
    }
    __syncthreads();
    fence_after();
    if (warp == 13) tmem_dealloc(tmem, 512);
}

// ---- single tokens: four CTAs per chain, a warp owns eight rows of the state, lane l columns 4 l .. 4 l + 3 of each ----
constexpr int kStepRows = 8, kStepSplit = 4;

__global__ void __launch_bounds__(128) linear_step_kernel(const __grid_constant__ LinearArgs a) {
    grid_dep_launch();
    grid_dep_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t chain = blockIdx.x / kStepSplit;
    const Chain ch = locate(a, chain);
    if (ch.len > 1) return;   // (the chunk kernel's)
    const int row0 = (warp * kStepSplit + (int)(blockIdx.x % kStepSplit)) * kStepRows;
    const int64_t at = (chain * kD + row0) * (int64_t)kD + lane * 4;
    float s[kStepRows][4];
    if (a.h0 == nullptr) {
#pragma unroll
        for (int r = 0; r < kStepRows; ++r) s[r][0] = s[r][1] = s[r][2] = s[r][3] = 0.0f;
    } else if (a.state_fp32) {
#pragma unroll
        for (int r = 0; r < kStepRows; ++r) {
            const float4 x = *reinterpret_cast<const float4*>(static_cast<const float*>(a.h0) + at + r * kD);
            s[r][0] = x.x; s[r][1] = x.y; s[r][2] = x.z; s[r][3] = x.w;
        }
    } else {
#pragma unroll
        for (int r = 0; r < kStepRows; ++r) {
            const uint2 x = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(a.h0) + at + r * kD);
            s[r][0] = bf_lo(x.x); s[r][1] = bf_hi(x.x); s[r][2] = bf_lo(x.y); s[r][3] = bf_hi(x.y);
        }
    }
    if (ch.len == 1) {
        const int hk = ch.h / a.group;
        const uint2 qr = *reinterpret_cast<const uint2*>(a.q + ch.b * a.q_batch + ch.t0 * a.q_token + hk * a.q_head + lane * 4);
        const uint2 kr = *reinterpret_cast<const uint2*>(a.k + ch.b * a.k_batch + ch.t0 * a.k_token + hk * a.k_head + lane * 4);
        const float decay = ex2_approx(log2_decay(a.g[ch.b * a.g_batch + ch.t0 * a.g_token + ch.h * a.g_head]));
        const __nv_bfloat16* vp = a.v + ch.b * a.v_batch + ch.t0 * a.v_token + ch.h * a.v_head + row0;
        const uint4 vr = *reinterpret_cast<const uint4*>(vp);
        const float q[4] = {bf_lo(qr.x), bf_hi(qr.x), bf_lo(qr.y), bf_hi(qr.y)}, k[4] = {bf_lo(kr.x), bf_hi(kr.x), bf_lo(kr.y), bf_hi(kr.y)};
        const float v[8] = {bf_lo(vr.x), bf_hi(vr.x), bf_lo(vr.y), bf_hi(vr.y), bf_lo(vr.z), bf_hi(vr.z), bf_lo(vr.w), bf_hi(vr.w)};
        float o[kStepRows];
#pragma unroll
        for (int r = 0; r < kStepRows; ++r) {
#pragma unroll
            for (int i = 0; i < 4; ++i) s[r][i] = __fmaf_rn(s[r][i], decay, v[r] * k[i]);
            o[r] = __fmaf_rn(s[r][3], q[3], __fmaf_rn(s[r][2], q[2], __fmaf_rn(s[r][1], q[1], s[r][0] * q[0])));
        }
        // sums over the warp: at each halving step a lane keeps half of the rows; lane l ends with row l / 4
#pragma unroll
        for (int off = 16; off >= 4; off >>= 1) {
            const bool up = (lane & off) != 0;
            const int rows = off / 4;
#pragma unroll
            for (int i = 0; i < rows; ++i) {
                const float send = up ? o[i] : o[i + rows], keep = up ? o[i + rows] : o[i];
                o[i] = keep + __shfl_xor_sync(0xffffffffu, send, off);
            }
        }
        o[0] += __shfl_xor_sync(0xffffffffu, o[0], 2);
        o[0] += __shfl_xor_sync(0xffffffffu, o[0], 1);
        if ((lane & 3) == 0) a.out[ch.b * a.out_batch + ch.t0 * a.out_token + ch.h * a.out_head + row0 + lane / 4] = f2bf(o[0] * a.scale);
    }
    if (a.hT == nullptr) return;
    if (a.state_fp32) {
#pragma unroll
        for (int r = 0; r < kStepRows; ++r)
            *reinterpret_cast<float4*>(static_cast<float*>(a.hT) + at + r * kD) = make_float4(s[r][0], s[r][1], s[r][2], s[r][3]);
    } else {
#pragma unroll
        for (int r = 0; r < kStepRows; ++r)
            *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.hT) + at + r * kD) = make_uint2(pack_bf2(s[r][0], s[r][1]), pack_bf2(s[r][2], s[r][3]));
    }
}

}  // namespace

size_t linear_workspace(const fkda_linear_params&) { return 0; }

int launch_linear(const fkda_linear_params& p, cudaStream_t stream, int* n_launches) {
    LinearArgs a;
    a.g = p.g;
    a.q = static_cast<__nv_bfloat16*>(const_cast<void*>(p.q));
    a.k = static_cast<__nv_bfloat16*>(const_cast<void*>(p.k));
    a.v = static_cast<__nv_bfloat16*>(const_cast<void*>(p.v));
    a.out = static_cast<__nv_bfloat16*>(p.out);
    a.h0 = p.initial_state;
    a.hT = p.final_state;
    a.cu = p.cu_seqlens;
    a.T = p.T; a.N = p.N;
    a.g_batch = p.g_stride[0]; a.g_token = p.g_stride[1]; a.g_head = p.g_stride[2];
    a.out_batch = p.out_stride[0]; a.out_token = p.out_stride[1]; a.out_head = p.out_stride[2];
    a.q_batch = p.q_stride[0]; a.q_token = p.q_stride[1]; a.q_head = p.q_stride[2];
    a.k_batch = p.k_stride[0]; a.k_token = p.k_stride[1]; a.k_head = p.k_stride[2];
    a.v_batch = p.v_stride[0]; a.v_token = p.v_stride[1]; a.v_head = p.v_stride[2];
    a.H = (int)p.H;
    a.group = (int)(p.H / p.Hk);
    a.scale = p.scale;
    a.state_fp32 = p.state_dtype == FKDA_STATE_FP32;
    const int64_t chains = p.N * p.H;
    if (chains > 0x7fffffff / kStepSplit) return FKDA_ERR_BAD_SHAPE;
    // single tokens: a fixed batch of them, or a packed batch that may hold many (the host sees only the totals): the step kernel then
    // serves the sequences of at most one token and the chunk kernel the others
    const bool single = p.cu_seqlens == nullptr ? p.T <= 1 : p.T < 2 * p.N;
    const bool chunks = p.cu_seqlens == nullptr ? p.T > 1 : p.T > 1;
    a.skip_single = single;
    int launches = 0;
    if (single) {
        if (!launch_dependent(linear_step_kernel, chains * kStepSplit, 128, 0, stream, a)) return FKDA_ERR_LAUNCH;
        ++launches;
    }
    if (chunks) {
        LinearMaps maps;
        auto map4 = [&](CUtensorMap* m, const void* base, int64_t heads, const int64_t* st) {
            const cuuint64_t dims[4] = {(cuuint64_t)kD, (cuuint64_t)heads, (cuuint64_t)p.T, (cuuint64_t)p.B};
            const cuuint64_t strides[3] = {(cuuint64_t)st[2] * 2, (cuuint64_t)st[1] * 2, (cuuint64_t)st[0] * 2};
            const cuuint32_t box[4] = {64u, 1u, (cuuint32_t)kC, 1u};
            return encode_bf16_map(m, 4, base, dims, strides, box);
        };
        if (!map4(&maps.q, p.q, p.Hk, p.q_stride) || !map4(&maps.k, p.k, p.Hk, p.k_stride) || !map4(&maps.v, p.v, p.H, p.v_stride))
            return FKDA_ERR_LAUNCH;
        if (!allow_smem<linear_chunk_kernel>(kSmem)) return FKDA_ERR_LAUNCH;
        if (!launch_dependent(linear_chunk_kernel, chains, kThreads, kSmem, stream, a, maps)) return FKDA_ERR_LAUNCH;
        ++launches;
    }
    *n_launches = launches;
    return FKDA_OK;
}

int linear_gave_up(cudaStream_t stream, int32_t* word) { return read_gave_up(stream, word); }

}  // namespace fkda
