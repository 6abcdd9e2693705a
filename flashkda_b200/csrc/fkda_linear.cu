// Linear attention with a decay for each head:
//     S_t = exp(g_t) S_{t-1} + v_t k_t^T  ([V, K]),   o_t = scale S_t q_t
//
// Prompts go through chunks of 64 tokens.  With G the running sum of g in a chunk and S the state in front of it,
//     O^T = scale (V^T P^T + S Q^T diag(exp(G))),   P_ij = exp(G_i - G_j) (q_i . k_j) for j <= i
//     S' = exp(G_64) S + (diag(w) V)^T K,           w_j = exp(G_64 - G_j)
// The call is bound by HBM (1 KB per token and head against 2 x 128 x (64 + 128 + 128) operations), so one CTA walks a (sequence,
// head) chain with everything between the copies in and out on the chip.  All products but q k^T have 128 rows (dimensions of v) on
// tcgen05: the fp32 state stays in tensor memory for the whole sequence, and what multiplies k and q there (weighted values, a bf16 copy
// of the state) is written to tensor memory as well, not through shared memory, whose bandwidth an earlier form with 64-row products
// ran out of.  A chunk's stages are spread over warpgroups: state (read, decayed, copied; in two halves, one of which is decayed
// while the other is updated), weights, outputs (two), weighted values (two), and a warp each for copies, two kinds of products and
// decays.  Seven warps per scheduler want small code: roles that were unrolled waited for instructions 44 % of the time, 3.4 us per chunk
// against 1.5 (96 chains) now.
// Measured: 148 chains of 8 192 tokens 236 us, 5.3 TB/s (0.80 of the copy bandwidth); 8 x 16 384 tokens of 64 heads (512 chains: 3.46 rounds
// of SMs, four are run) 1.66 ms, 1.79 to 1.92 where the power cap holds the clock (1.6 to 1.75 GHz); a chain alone 1.5 us per chunk, which is the loop
// from one update of the state to the next.  Few long chains are cut into segments (see plan()): 32 chains of 8 192 tokens 104 us, in one
// piece 205.
//
// Numerics: decays are sums of g in fp32 over at most 64 tokens, w as sums over the tokens behind j (no differences of large sums).
// P and the copy of S that Q multiplies are operands of products and rounded to bf16 for them: bf16 outputs are 2.35e-3 from 64 bits
// (2-norm), where their own rounding alone is 1.66e-3.  The state is not rounded: it is fp32 throughout, and w V enters the product as three bf16 terms, which hold all 24 bits; as two, which hold 16, where the
// initial state is bf16 (half a step of its own is 2^-8, of the terms 2^-16; 6 % less time where the power cap rules).  The tensor cores
// cut fp32 sums off where an addition elsewhere would round, twelve times a chunk, so an fp32 state comes out low by what its memory
// gathers: 1.3e-7 of it for decays of exp(-1), 4e-7 for exp(-1/64), 1.3e-6 for exp(-1/256), 4.5e-6 for exp(-1/1024), 2.7e-5 for
// exp(-1/8192) over 16 384 tokens.
//
// Single tokens: a read-modify-write of the state by a kernel of its own, as bound by HBM as that is (256 x 64 states in bf16: 172 to
// 190 us, 0.97 to 0.87 of the copy bandwidth; one sequence: the launch, 2.6 to 3.2 us).  Of a packed batch the host does not know that all
// sequences are such, and the chunk kernel's CTAs, one to an SM, have to come and see: 294 us for the same 256 x 64 states.
#include "fkda_tc5.cuh"

namespace fkda {
namespace {

using namespace tc5;

constexpr int kC = 64;                        // tokens of a chunk
constexpr int kTileBytes = kC * 128;          // 64 tokens x 64 dimensions
constexpr int kOperandBytes = 2 * kTileBytes; // a chunk of q, k or v
constexpr int kStageBytes = 3 * kOperandBytes;
constexpr int kStages = 3;
constexpr int kThreads = 896;                 // warpgroups: one each for state and scores, two each for outputs and values; copies, products, decays
constexpr int kOffP = kStages * kStageBytes;
constexpr int kOffOut = kOffP + 2 * kTileBytes;
constexpr int kOffBars = kOffOut + 2 * kOperandBytes;
// Tensor-memory columns: the state, its bf16 copy, scores, the two parts of the outputs, the weighted values' terms
constexpr uint32_t kS = 0, kCopy = 128, kScore = 192, kO1 = 256, kO2 = 320, kW = 384;

constexpr int kMaxOrdered = 64;               // packed sequences that are taken in the order of their lengths
static_assert(kMaxOrdered <= kThreads, "a thread ranks a sequence");

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
    bool state_fp32;
    bool skip_single;       // the chunk kernel leaves sequences of at most one token to the step kernel (packed, no segments, not ordered)
    bool ordered;           // packed sequences: the longest first
    int seg_len, seg_rows;  // tokens of a segment, 0: every chain is walked in one piece; rows that the workspace has
    float* seg_state;       // [segment][head][128][128], and behind them
    float* seg_decay;       // [segment][head]
    int starve_ms;          // test hook: nothing is loaded, and a wait gives up after so long
};
struct LinearMaps {
    CUtensorMap q, k, v, out;
};
struct Decays {
    alignas(16) float G[kC], eG[kC], w[kC], total;
    float pad[3];
};
// (A barrier that one side may complete twice before the other has looked is there once per buffer.)
struct Bars {
    Decays decay[kStages];
    uint64_t full[kStages], empty[kStages], dec_full[kStages], dec_empty[kStages], score, score_free, p_full[2], p_free[2], out_full, out_free, scaled[2], s_done[2], copy_free,
        w_full[2], drained[2];
    uint32_t tmem;
    int abort, chosen;
};
constexpr int kSmem = kOffBars + ((int)sizeof(Bars) + 127) / 128 * 128;
static_assert(kSmem <= 232448, "shared memory of an SM");

constexpr float kLog2e = 1.4426950408889634f;
// exp(-100) is nothing in fp32; a decay below it (minus infinity to start afresh) would make differences of sums meaningless.
__device__ __forceinline__ float log2_decay(float g) { return (g < -100.0f ? -100.0f : g) * kLog2e; }

// What a CTA walks: a sequence's head, or one segment of it.
struct Chain {
    int64_t n, b, t0;      // sequence, batch row, first token
    int h, len;
    int seg, segs;         // segment of the sequence's, of which there are `segs`
    int64_t slot;          // of the segment and head in the workspace
};
__device__ __forceinline__ int seq_len(const LinearArgs& a, int64_t n, int64_t* first) {
    const int64_t lo = a.cu[n] < 0 ? 0 : a.cu[n], hi = a.cu[n + 1] > a.T ? a.T : a.cu[n + 1];
    *first = lo;
    return hi > lo ? (int)(hi - lo) : 0;
}
__device__ __forceinline__ int segments(const LinearArgs& a, int len) { return a.seg_len == 0 || len == 0 ? 1 : (len + a.seg_len - 1) / a.seg_len; }
// (Not inlined, nor is the next one: inlined, such searches made the products slower, as they did in the prompts' kernel; probably the
// compiler no longer knows then that the warps are converged.)
// `row`: of (sequence, segment) pairs in order; len < 0: there are fewer.
__device__ __noinline__ Chain locate(const LinearArgs& a, int64_t row, int h) {
    Chain c;
    c.h = h;
    c.slot = row * a.H + h;
    c.b = 0;
    c.seg = 0;
    c.segs = 1;
    if (a.cu == nullptr) {
        c.segs = segments(a, (int)a.T);
        c.n = c.segs == 1 ? row : row / c.segs;
        c.seg = (int)(row - c.n * c.segs);
        c.b = c.n;
        c.t0 = 0;
        c.len = c.n < a.N ? (int)a.T : -1;
    } else if (a.seg_len == 0) {
        c.n = row;
        c.len = row < a.N ? seq_len(a, row, &c.t0) : -1;
    } else {   // (few sequences)
        int64_t seen = 0;
        c.len = -1;
        for (c.n = 0; c.n < a.N; ++c.n) {
            const int len = seq_len(a, c.n, &c.t0);
            c.segs = segments(a, len);
            if (row < seen + c.segs) {
                c.seg = (int)(row - seen);
                if (seen + c.segs <= a.seg_rows) c.len = len;   // (always, unless cu_seqlens runs backwards)
                break;
            }
            seen += c.segs;
        }
    }
    if (c.len > 0 && c.segs > 1) {
        c.t0 += (int64_t)c.seg * a.seg_len;
        c.len = min(a.seg_len, c.len - c.seg * a.seg_len);
    }
    return c;
}

// The sequence that `row` others come before: by length, then by number.
__device__ __noinline__ void in_order(const LinearArgs& a, int row, int* lens, int* chosen) {
    int64_t first;
    const int me = threadIdx.x, len = me < a.N ? seq_len(a, me, &first) : 0;
    if (me < a.N) lens[me] = len;
    fence_proxy_async_smem();
    __syncthreads();
    int rank = 0;
    if (me < a.N)
#pragma unroll 1
        for (int i = 0; i < (int)a.N; ++i) rank += lens[i] > len || (lens[i] == len && i < me) ? 1 : 0;
    if (me < a.N && rank == row) *chosen = me;
    fence_proxy_async_smem();
    __syncthreads();
}

// 32 numbers of a row of a state
__device__ __forceinline__ void load_state32(const void* from, bool fp32, int64_t at, uint32_t* r) {
    if (from == nullptr) {
#pragma unroll
        for (int i = 0; i < 32; ++i) r[i] = 0u;
    } else if (fp32) {
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const float*>(from) + at);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint4 x = src[i];
            r[4 * i] = x.x; r[4 * i + 1] = x.y; r[4 * i + 2] = x.z; r[4 * i + 3] = x.w;
        }
    } else {
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(from) + at);
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
__device__ __forceinline__ void store_state32(void* to, bool fp32, int64_t at, const uint32_t* r) {
    if (fp32) {
        uint4* dst = reinterpret_cast<uint4*>(static_cast<float*>(to) + at);
#pragma unroll
        for (int i = 0; i < 8; ++i) dst[i] = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
    } else {
        uint4* dst = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(to) + at);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            dst[i] = make_uint4(pack_bf2(f(r[8 * i]), f(r[8 * i + 1])), pack_bf2(f(r[8 * i + 2]), f(r[8 * i + 3])),
                                pack_bf2(f(r[8 * i + 4]), f(r[8 * i + 5])), pack_bf2(f(r[8 * i + 6]), f(r[8 * i + 7])));
    }
}

// kStates: only the state that each segment but the last leaves behind a zero one (the first: behind the initial state), and the
// product of its decays.  kTerms: of the weighted values, 2 where the initial state is bf16, else 3.
template <bool kStates, int kTerms>
__global__ void __launch_bounds__(kThreads, 1) linear_chunk_kernel(const __grid_constant__ LinearArgs a, const __grid_constant__ LinearMaps maps) {
    extern __shared__ __align__(1024) uint8_t smem[];
    Bars& bar = *reinterpret_cast<Bars*>(smem + kOffBars);
    if (a.skip_single) {   // (before anything is set up: most CTAs find nothing to do)
        grid_dep_launch();
        grid_dep_wait();
        int64_t first;
        if (seq_len(a, blockIdx.x / (uint32_t)a.H, &first) <= 1) return;
    }
    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) mbar_init(&bar.full[i], 1), mbar_init(&bar.empty[i], kStates ? 1 : 2), mbar_init(&bar.dec_full[i], 1), mbar_init(&bar.dec_empty[i], kStates ? 12 : 24);
        for (int i = 0; i < 2; ++i) mbar_init(&bar.p_full[i], 128), mbar_init(&bar.p_free[i], 1), mbar_init(&bar.w_full[i], 128);
        mbar_init(&bar.score, 1);
        mbar_init(&bar.score_free, 128);
        mbar_init(&bar.out_full, 1);
        mbar_init(&bar.out_free, 256);
        for (int i = 0; i < 2; ++i) mbar_init(&bar.scaled[i], 128), mbar_init(&bar.s_done[i], 1);
        mbar_init(&bar.copy_free, 1);
        for (int i = 0; i < 2; ++i) mbar_init(&bar.drained[i], 1);
        bar.abort = 0;
        mbar_fence_init();
    }
    if (warp == 25) tmem_alloc(&bar.tmem, 512);
    fence_before();
    grid_dep_launch();
    grid_dep_wait();
    __syncthreads();
    fence_after();
    constexpr uint32_t tmem = 0;   // (all columns are this CTA's)
    int row = (int)(blockIdx.x / (uint32_t)a.H);
    if (a.ordered) {   // the sequence that as many others come before as rows are in front of mine
        in_order(a, row, reinterpret_cast<int*>(smem), &bar.chosen);
        row = bar.chosen;
    }
    const Chain ch = locate(a, row, (int)(blockIdx.x % (uint32_t)a.H));
    const bool last = ch.seg + 1 == ch.segs;
    const bool mine = ch.len >= 0 && !(kStates && last) && as_assumed(smem, bar.tmem);
    const int n = uniform(mine ? (ch.len + kC - 1) / kC : 0);

    if (warp == 24) {
        // ---- copies ----
        const uint32_t base = smem_u32(smem), leader = elect_one();
        const int t0 = uniform((int)ch.t0), row = uniform((int)ch.b), head = uniform(ch.h), key_head = uniform(ch.h / a.group);
        int c = 0, stage = 0, phase = 1;
        if (a.starve_ms > 0) starve(&bar.full[0], a.starve_ms, &bar.abort), c = n;
#pragma unroll 1
        for (; c < n; ++c) {
            if (c >= kStages && !__all_sync(0xffffffffu, wait_free(&bar.empty[stage], phase, &bar.abort))) break;
            const uint32_t dst = base + stage * kStageBytes;
            expect(&bar.full[stage], kStates ? 2 * kOperandBytes : kStageBytes, leader);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                if (!kStates) load_4d(dst + x * kTileBytes, &maps.q, x * 64, key_head, t0 + c * kC, row, &bar.full[stage], leader);
                load_4d(dst + kOperandBytes + x * kTileBytes, &maps.k, x * 64, key_head, t0 + c * kC, row, &bar.full[stage], leader);
                load_4d(dst + 2 * kOperandBytes + x * kTileBytes, &maps.v, x * 64, head, t0 + c * kC, row, &bar.full[stage], leader);
            }
            if (++stage == kStages) stage = 0, phase ^= 1;
        }
#pragma unroll 1
        for (int k = a.starve_ms > 0 ? c : max(0, c - kStages); k < c; ++k) drain(&bar.full[k % kStages], (k / kStages) & 1);
        __syncwarp();
    } else if (warp == 25) {
        // ---- products of the state, which the next chunk waits for, and scores ----
        if (n > 0) {
            const uint32_t base = smem_u32(smem), leader = elect_one();
            constexpr uint32_t kIdScore = idesc(64, 64, false, false), kIdState = idesc(128, 64, false, true);
            int stage = 0, phase = 0;   // of the chunk whose scores are next
            uint32_t k = 0;             // keys of the chunk in front of it
#pragma unroll 1
            for (int c = -1; c < n; ++c) {
                if (c >= 0) {
#pragma unroll 1
                    for (int h = 0; h < 2; ++h) {   // 64 columns of the state, while the other 64 are being decayed
                        wait_warp(&bar.scaled[h], c & 1, &bar.abort);
                        wait_warp(&bar.w_full[0], c & 1, &bar.abort);
                        wait_warp(&bar.w_full[1], c & 1, &bar.abort);
                        fence_after();
#pragma unroll 1
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int t = 0; t < kTerms; ++t)
                                mma_ts(tmem + kS + h * 64, tmem + kW + t * 32 + i * 8, k + h * (kTileBytes / 16) + i * (2048 / 16), kIdState, 1, leader);
                        commit(&bar.s_done[h], leader);
                    }
                    commit(&bar.empty[stage == 0 ? kStages - 1 : stage - 1], leader);
                }
                if (c + 1 < n) {
                    wait_warp(&bar.full[stage], phase, &bar.abort);
                    k = desc(base + stage * kStageBytes + kOperandBytes);
                    if (!kStates) {
                    if (c >= 0) wait_warp(&bar.score_free, c & 1, &bar.abort);
                    fence_after();
                    const uint32_t q = desc(base + stage * kStageBytes);
#pragma unroll 1
                    for (int x = 0; x < 2; ++x)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            mma_ss(tmem + kScore, q + x * (kTileBytes / 16) + i * 2, k + x * (kTileBytes / 16) + i * 2, kIdScore, (x | i) != 0, leader);
                    commit(&bar.score, leader);
                    }
                    if (++stage == kStages) stage = 0, phase ^= 1;
                }
            }
            commit(&bar.drained[0], leader);
            drain(&bar.drained[0], 0);
        }
    } else if (warp == 27) {
        // ---- products of the outputs ----
        if (n > 0 && !kStates) {
            const uint32_t base = smem_u32(smem), leader = elect_one();
            constexpr uint32_t kIdO1 = idesc(128, 64, false, false), kIdO2 = idesc(128, 64, true, false);
            int stage = 0, phase = 0;
#pragma unroll 1
            for (int c = 0; c < n; ++c) {
                const uint32_t q = desc(base + stage * kStageBytes), v = desc(base + stage * kStageBytes + 2 * kOperandBytes, kTileBytes);
                wait_warp(&bar.full[stage], phase, &bar.abort);
                wait_warp(&bar.scaled[1], c & 1, &bar.abort);   // (the copy is there as well)
                if (c > 0) wait_warp(&bar.out_free, (c - 1) & 1, &bar.abort);
                fence_after();
#pragma unroll 1
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        mma_ts(tmem + kO1, tmem + kCopy + x * 32 + i * 8, q + (x * kTileBytes + i * 32) / 16, kIdO1, (x | i) != 0, leader);
                commit(&bar.copy_free, leader);
                if (c + 1 == n) wait_warp(&bar.w_full[1], c & 1, &bar.abort);   // (values behind the sequence's end are nothing by now)
                wait_warp(&bar.p_full[c & 1], (c >> 1) & 1, &bar.abort);
                fence_after();
                const uint32_t p = desc(base + kOffP + (c & 1) * kTileBytes);
#pragma unroll
                for (int i = 0; i < 4; ++i) mma_ss(tmem + kO2, v + i * 2048 / 16, p + i * 32 / 16, kIdO2, i != 0, leader);
                commit(&bar.p_free[c & 1], leader);
                commit(&bar.out_full, leader);
                commit(&bar.empty[stage], leader);
                if (++stage == kStages) stage = 0, phase ^= 1;
            }
            commit(&bar.drained[1], leader);
            drain(&bar.drained[1], 0);
        }
    } else if (warp == 26) {
        // ---- decays: lane l has tokens 2 l and 2 l + 1 of a chunk ----
        float all = 0.0f;
        const float* g = a.g + ch.b * a.g_batch + ch.t0 * a.g_token + ch.h * a.g_head;
#pragma unroll 1
        for (int c = 0; c < n; ++c) {
            const int t = c * kC + 2 * lane;
            const float x = t < ch.len ? log2_decay(g[t * a.g_token]) : 0.0f, y = t + 1 < ch.len ? log2_decay(g[(t + 1) * a.g_token]) : 0.0f;
            float upto = x + y, from = x + y;   // sums over the lanes up to mine, and from mine on
#pragma unroll 1
            for (int off = 1; off < 32; off <<= 1) {
                const float p = __shfl_up_sync(0xffffffffu, upto, off), q = __shfl_down_sync(0xffffffffu, from, off);
                if (lane >= off) upto += p;
                if (lane + off < 32) from += q;
            }
            const float before = __shfl_up_sync(0xffffffffu, upto, 1), behind = __shfl_down_sync(0xffffffffu, from, 1);
            const float G0 = (lane > 0 ? before : 0.0f) + x, G1 = G0 + y, w1 = lane < 31 ? behind : 0.0f, w0 = w1 + y;
            if (c >= kStages) wait_warp(&bar.dec_empty[c % kStages], (c / kStages - 1) & 1, &bar.abort);
            Decays& d = bar.decay[c % kStages];
            *reinterpret_cast<float2*>(&d.G[2 * lane]) = make_float2(G0, G1);
            *reinterpret_cast<float2*>(&d.eG[2 * lane]) = make_float2(ex2_approx(G0) * a.scale, ex2_approx(G1) * a.scale);
            *reinterpret_cast<float2*>(&d.w[2 * lane]) = make_float2(ex2_approx(w0), ex2_approx(w1));
            if (lane == 0) d.total = ex2_approx(from);
            all += from;
            __syncwarp();
            if (lane == 0) arrive(&bar.dec_full[c % kStages]);
        }
        if (kStates && n > 0 && lane == 0) a.seg_decay[ch.slot] = ex2_approx(all);
    } else if (warp < 4) {
        // ---- state: thread = row (dimension of v); decayed in place, with a bf16 copy of what it was for the product with q ----
        const int v = warp * 32 + lane;
        const uint32_t lanes = (uint32_t)(warp * 32) << 16, ts = tmem + kS + lanes;
        const int64_t at = ((ch.n * a.H + ch.h) * kD + v) * (int64_t)kD, seg_at = (ch.slot * kD + v) * (int64_t)kD;
        // the state in front: the call's, a copy of it (its buffer may be the final state's, which the last segment writes while the first
        // one starts), or what the segment in front leaves
        const void* from = a.h0;
        bool fp32 = a.state_fp32;
        int64_t from_at = at;
        if (kStates && ch.seg > 0 && !last) from = nullptr;
        if (!kStates && ch.segs > 1 && (ch.seg > 0 || a.h0 != nullptr)) {
            from = a.seg_state;
            fp32 = true;
            from_at = seg_at + (int64_t)(ch.seg > 0 ? -1 : ch.segs - 1) * a.H * (kD * kD);
        }
        if (n > 0) {
#pragma unroll 1
            for (int x = 0; x < 4; ++x) {
                uint32_t r[32];
                load_state32(from, fp32, from_at + x * 32, r);
                st32(ts + x * 32, r);
            }
            wait_st();
        }
#pragma unroll 1
        for (int c = 0; c < n; ++c) {
            const int s = c % kStages;
            wait_warp(&bar.dec_full[s], (c / kStages) & 1, &bar.abort);
            const float total = bar.decay[s].total;
            __syncwarp();
            mbar_arrive_lane0(&bar.dec_empty[s], lane);
            if (!kStates && c > 0) wait_warp(&bar.copy_free, (c - 1) & 1, &bar.abort);
#pragma unroll 1
            for (int h = 0; h < 2; ++h) {
                if (c > 0) {
                    wait_warp(&bar.s_done[h], (c - 1) & 1, &bar.abort);
                    fence_after();
                }
#pragma unroll 1
                for (int x = 2 * h; x < 2 * h + 2; ++x) {
                    uint32_t r[32], copy[16];
                    ld32(ts + x * 32, r);
                    wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        copy[i] = pack_bf2(f(r[2 * i]), f(r[2 * i + 1]));
                        mul2(r[2 * i], r[2 * i + 1], total, total);
                    }
                    st32(ts + x * 32, r);
                    if (!kStates) st16(tmem + kCopy + lanes + x * 16, copy);
                }
                wait_st();
                fence_before();
                arrive(&bar.scaled[h]);
            }
        }
        if (n > 0) {
            wait_warp(&bar.s_done[0], (n - 1) & 1, &bar.abort);
            wait_warp(&bar.s_done[1], (n - 1) & 1, &bar.abort);
            fence_after();
        }
        const bool keeps = kStates ? ch.len >= 0 && ch.segs > 1 && (!last || a.h0 != nullptr) : mine && last && a.hT != nullptr;
        if (keeps) {
#pragma unroll 1
            for (int x = 0; x < 4; ++x) {
                uint32_t r[32];
                if (n > 0) {
                    ld32(ts + x * 32, r);
                    wait_ld();
                } else {   // (an empty sequence, or the copy of the initial state in the last segment's place)
                    load_state32(from, fp32, from_at + x * 32, r);
                }
                if (kStates) store_state32(a.seg_state, true, seg_at + x * 32, r);
                else store_state32(a.hT, a.state_fp32, at + x * 32, r);
            }
        }
        fence_before();
    } else if (warp < 8) {
        // ---- scores to weights: warp w has rows (queries) 16 w .. 16 w + 15, thread 4 g + t rows g and g + 8 of these ----
        if (!kStates) {
        const int w = warp - 4, gr = lane >> 2, tc = lane & 3;
        const int r0 = w * 16 + gr, r1 = r0 + 8;
#pragma unroll 1
        for (int c = 0; c < n; ++c) {
            wait_warp(&bar.dec_full[c % kStages], (c / kStages) & 1, &bar.abort);
            const Decays& d = bar.decay[c % kStages];
            const float G0 = d.G[r0], G1 = d.G[r1];
            if (c >= 2) wait_warp(&bar.p_free[c & 1], (c / 2 - 1) & 1, &bar.abort);
            wait_warp(&bar.score, c & 1, &bar.abort);
            fence_after();
            uint8_t* p = smem + kOffP + (c & 1) * kTileBytes + r0 * 128 + tc * 4;   // (r1 = r0 + 8 has the same swizzle)
#pragma unroll 1
            for (int b = 0; b < 4; ++b) {   // 16 columns; those behind the warp's last row are masked for all of its rows
                uint32_t s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                if (b <= w) {
                    ld_frag16(tmem + kScore + b * 16 + ((uint32_t)(w * 32) << 16), s);
                    wait_ld();
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int j = b * 16 + 8 * i + 2 * tc;
                        const float2 G = *reinterpret_cast<const float2*>(&d.G[j]);
                        s[4 * i] = j <= r0 ? u(f(s[4 * i]) * ex2_approx(G0 - G.x)) : 0u;
                        s[4 * i + 1] = j < r0 ? u(f(s[4 * i + 1]) * ex2_approx(G0 - G.y)) : 0u;
                        s[4 * i + 2] = j <= r1 ? u(f(s[4 * i + 2]) * ex2_approx(G1 - G.x)) : 0u;
                        s[4 * i + 3] = j < r1 ? u(f(s[4 * i + 3]) * ex2_approx(G1 - G.y)) : 0u;
                    }
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int unit = ((2 * b + i) ^ gr) << 4;
                    *reinterpret_cast<uint32_t*>(p + unit) = pack_bf2(f(s[4 * i]), f(s[4 * i + 1]));
                    *reinterpret_cast<uint32_t*>(p + 8 * 128 + unit) = pack_bf2(f(s[4 * i + 2]), f(s[4 * i + 3]));
                }
            }
            fence_before();
            arrive(&bar.score_free);
            fence_proxy_async_smem();
            arrive(&bar.p_full[c & 1]);
            __syncwarp();
            mbar_arrive_lane0(&bar.dec_empty[c % kStages], lane);
        }
        }
    } else if (warp < 16) {
        // ---- outputs: fragments of 16 dimensions of v x 32 tokens, stored transposed as rows of tokens, which one copy takes away (or the
        //      warps themselves, where the chunk's last rows are not the sequence's) ----
        if (!kStates) {
        const int w = warp & 3, half = (warp - 8) >> 2, tc = lane & 3, me = threadIdx.x & 255;   // a warpgroup has 32 of the tokens
        // the lane's row address within four 8 x 8 blocks (two of tokens x two of dimensions)
        const int token = (lane & 7) + ((lane >> 4) << 3), unit = (w & 1) * 4 + ((lane >> 3) & 1);
        const uint32_t tile = smem_u32(smem) + kOffOut + (w >> 1) * kTileBytes + token * 128;
#pragma unroll 1
        for (int c = 0; c < n; ++c) {
            const Decays& d = bar.decay[c % kStages];
            const uint32_t buffer = tile + (c & 1) * kOperandBytes;
            const int valid = ch.len - c * kC;
            if (me == 0) bulk_wait_group_read<1>();   // (the copy that the buffer's last outputs went with)
            wait_warp(&bar.dec_full[c % kStages], (c / kStages) & 1, &bar.abort);
            named_sync(2, 256);
            wait_warp(&bar.out_full, c & 1, &bar.abort);
            fence_after();
#pragma unroll 1
            for (int up = 0; up < 2; ++up) {   // 16 of the warp's dimensions
                const uint32_t lanes = (uint32_t)(w * 32 + up * 16) << 16;
                uint32_t o1[16], o2[16];
                ld_frag32(tmem + kO1 + half * 32 + lanes, o1);
                ld_frag32(tmem + kO2 + half * 32 + lanes, o2);
                wait_ld();
                const uint32_t row = buffer + half * 32 * 128 + (((unit + 2 * up) ^ (lane & 7)) << 4);
#pragma unroll
                for (int i = 0; i < 2; ++i) {   // 16 tokens
                    uint32_t y[4];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float2 e = *reinterpret_cast<const float2*>(&d.eG[half * 32 + i * 16 + j * 8 + 2 * tc]);
                        const uint32_t *p1 = o1 + 8 * i + 4 * j, *p2 = o2 + 8 * i + 4 * j;
                        y[2 * j] = pack_bf2(__fmaf_rn(f(p1[0]), e.x, f(p2[0]) * a.scale), __fmaf_rn(f(p1[1]), e.y, f(p2[1]) * a.scale));
                        y[2 * j + 1] = pack_bf2(__fmaf_rn(f(p1[2]), e.x, f(p2[2]) * a.scale), __fmaf_rn(f(p1[3]), e.y, f(p2[3]) * a.scale));
                    }
                    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(row + i * 16 * 128), "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3]) : "memory");
                }
            }
            fence_before();
            arrive(&bar.out_free);
            fence_proxy_async_smem();
            named_sync(2, 256);
            mbar_arrive_lane0(&bar.dec_empty[c % kStages], lane);
            if (valid >= kC) {
                if (me == 0) {
                    const uint8_t* src = smem + kOffOut + (c & 1) * kOperandBytes;
                    for (int x = 0; x < 2; ++x) tma_store_4d(&maps.out, x * 64, ch.h, (int)ch.t0 + c * kC, (int)ch.b, src + x * kTileBytes);
                    bulk_commit_group();
                }
            } else {
                __nv_bfloat16* out = a.out + ch.b * a.out_batch + (ch.t0 + c * kC) * a.out_token + ch.h * a.out_head;
#pragma unroll 1
                for (int i = me; i < valid * 16; i += 256) {
                    const int t = i >> 4, x = i & 15;
                    *reinterpret_cast<uint4*>(out + t * a.out_token + x * 8) =
                        *reinterpret_cast<const uint4*>(smem + kOffOut + (c & 1) * kOperandBytes + (x >> 3) * kTileBytes + t * 128 + (((x ^ t) & 7) << 4));
                }
            }
        }
        if (me == 0) bulk_wait_group<0>();
        }
    } else {
        // ---- weighted values: transposed reads give thread 4 g + t of warp w the token pairs 8 b + 2 t, + 1 of dimensions g, g + 8, g + 16
        //      and g + 24 of the warp's 32, as the A operand wants them; what is behind the sequence's end becomes nothing ----
        const int w = warp & 3, half = (warp - 16) >> 2, tc = lane & 3;   // a warpgroup has 32 of the tokens
        // the lane's row address within a group of four 8 x 8 blocks (two of tokens x two of dimensions)
        const int token = (lane & 7) + ((lane >> 4) << 3);            // of 16
        const int unit = (w & 1) * 4 + ((lane >> 3) & 1);               // 16-byte piece of the tile's row, + 2 for the upper 16 dimensions
        const uint32_t tile = smem_u32(smem) + 2 * kOperandBytes + (w >> 1) * kTileBytes + token * 128;
        const uint32_t piece[2] = {tile + ((unit ^ (lane & 7)) << 4), tile + (((unit + 2) ^ (lane & 7)) << 4)};
        const uint32_t tw = tmem + kW + ((uint32_t)(w * 32) << 16);
#pragma unroll 1
        for (int c = 0; c < n; ++c) {
            const int s = c % kStages, valid = ch.len - c * kC;
            wait_warp(&bar.dec_full[s], (c / kStages) & 1, &bar.abort);
            wait_warp(&bar.full[s], (c / kStages) & 1, &bar.abort);
            if (valid < kC) {
                uint8_t* k = smem + s * kStageBytes + kOperandBytes;
#pragma unroll 1
                for (int i = threadIdx.x & 255; i < (kC - valid) * 8; i += 256)
#pragma unroll
                    for (int x = 0; x < 4; ++x) *reinterpret_cast<uint4*>(k + x * kTileBytes + valid * 128 + i * 16) = make_uint4(0, 0, 0, 0);
                fence_proxy_async_smem();
                named_sync(1, 256);
            }
            uint32_t term[2][2][kTerms][4];
#pragma unroll
            for (int b = 0; b < 2; ++b) {          // 16 tokens
                const float *w0 = &bar.decay[s].w[half * 32 + b * 16 + 2 * tc], *w1 = w0 + 8;
#pragma unroll
                for (int d = 0; d < 2; ++d) {      // 16 dimensions
                    uint32_t r[4];
                    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(piece[d] + s * kStageBytes + (2 * half + b) * 2048) : "memory");
#pragma unroll
                    for (int i = 0; i < 4; ++i) {   // r[0], r[1]: tokens 0 .. 7, dimensions 0 .. 7 and 8 .. 15; r[2], r[3]: tokens 8 .. 15
                        uint32_t x = r[i] << 16, y = r[i] & 0xffff0000u;
                        mul2(x, y, i < 2 ? w0[0] : w1[0], i < 2 ? w0[1] : w1[1]);
#pragma unroll
                        for (int m = 0; m < kTerms; ++m) {
                            // the upper 16 bits of what is left, which are a bf16 (after three times nothing is left); the last one rounded
                            term[b][d][m][i] = m + 1 < kTerms ? __byte_perm(x, y, 0x7632) : pack_bf2(f(x), f(y));
                            if (m + 1 < kTerms) sub2(x, y, x & 0xffff0000u, y & 0xffff0000u);
                        }
                    }
                }
            }
            if (c > 0) {
                wait_warp(&bar.s_done[1], (c - 1) & 1, &bar.abort);   // (the last chunk's terms have been read)
                fence_after();
            }
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int d = 0; d < 2; ++d)
#pragma unroll
                    for (int m = 0; m < kTerms; ++m)
                        st_frag8(tw + m * 32 + (2 * half + b) * 8 + ((uint32_t)(d * 16) << 16), term[b][d][m][0], term[b][d][m][1], term[b][d][m][2], term[b][d][m][3]);
            wait_st();
            fence_before();
            arrive(&bar.w_full[half]);
            __syncwarp();
            mbar_arrive_lane0(&bar.dec_empty[s], lane);
        }
    }
    __syncthreads();
    fence_after();
    if (warp == 25) tmem_dealloc(tmem, 512);
}

// ---- single tokens: four CTAs per chain, a warp owns eight rows of the state, lane l columns 4 l .. 4 l + 3 of each ----
constexpr int kStepRows = 8, kStepSplit = 4;

__global__ void __launch_bounds__(128) linear_step_kernel(const __grid_constant__ LinearArgs a) {
    grid_dep_launch();
    grid_dep_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t chain = blockIdx.x / kStepSplit;
    Chain ch;
    ch.n = chain / (uint32_t)a.H;
    ch.h = (int)(chain % (uint32_t)a.H);
    ch.b = a.cu == nullptr ? ch.n : 0;
    ch.t0 = 0;
    ch.len = a.cu == nullptr ? (int)a.T : seq_len(a, ch.n, &ch.t0);
    if (ch.len > 1) return;   // (the chunk kernel's)
    const int row0 = (warp * kStepSplit + (int)(blockIdx.x % kStepSplit)) * kStepRows;
    const int64_t at = ((int64_t)chain * kD + row0) * kD + lane * 4;
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

// The states in front of the segments: what a segment left behind a zero state, plus what came in, decayed by it.  A CTA: a sixteenth
// of a chain's states, a float4 per thread.
__global__ void __launch_bounds__(256) linear_carry_kernel(const __grid_constant__ LinearArgs a) {
    grid_dep_launch();
    grid_dep_wait();
    const int64_t chain = blockIdx.x / 16, n = chain / a.H;
    int64_t row = 0, first;
    int segs = segments(a, (int)a.T);
    if (a.cu == nullptr) {
        row = n * segs;
    } else {
        for (int64_t i = 0; i < n; ++i) row += segments(a, seq_len(a, i, &first));
        segs = segments(a, seq_len(a, n, &first));
    }
    if (row + segs > a.seg_rows) return;
    const int64_t slot = row * a.H + chain % a.H;
    float4* at = reinterpret_cast<float4*>(a.seg_state) + slot * (kD * kD / 4) + (blockIdx.x % 16) * 256 + threadIdx.x;
    const int64_t step = (int64_t)a.H * (kD * kD / 4);
    float4 x = *at;
#pragma unroll 4
    for (int s = 1; s + 1 < segs; ++s) {
        const float decay = a.seg_decay[slot + (int64_t)s * a.H];
        float4 y = at[s * step];
        y.x = __fmaf_rn(decay, x.x, y.x);
        y.y = __fmaf_rn(decay, x.y, y.y);
        y.z = __fmaf_rn(decay, x.z, y.z);
        y.w = __fmaf_rn(decay, x.w, y.w);
        at[s * step] = y;
        x = y;
    }
}

template <bool kStates, int kTerms>
bool launch_walk(int64_t ctas, cudaStream_t stream, const LinearArgs& a, const LinearMaps& maps) {
    constexpr auto kKernel = linear_chunk_kernel<kStates, kTerms>;
    return allow_smem<kKernel>(kSmem) && launch_dependent(kKernel, ctas, kThreads, kSmem, stream, a, maps);
}

// Tokens of a segment, 0 for none, and how many (sequence, segment) rows there are at most.  Segments put the idle SMs of few long
// chains to work, for half of a chunk's work more: the states are made first, without outputs.
struct Segments {
    int len;
    int64_t rows;
};
Segments plan(const fkda_linear_params& p) {
    const Segments none{0, p.N};
    const int sms = device_sm_count();
    const bool packed = p.cu_seqlens != nullptr;
    const int64_t rows = sms / p.H - (packed ? p.N : 0);   // (every packed sequence has one that is not full)
    const int64_t pieces = packed ? rows : rows / p.N, tokens = p.T;
    if (pieces < 2 || p.N > 64 || tokens == 0) return none;
    const int64_t len = ((tokens + pieces - 1) / pieces + kC - 1) / kC * kC;
    const int64_t segs = (tokens + len - 1) / len;
    if (segs < 2) return none;
    // in units of a chunk of the whole walk: one with states only takes about 0.7, the two more launches and starts 8.  (Of a packed batch
    // only the tokens are known: its longest sequence is taken to have 2 / (N + 1) of them.)  Segments against one piece: 8 000 tokens of 1
    // head 58 us against 164, of 32 heads 102 against 173, 48 heads 129 against 168; 1 600 tokens of 32 heads 38.6 against 42.6, 1 200 34.1
    // against 34.7; at the line 2 x 4 000 of 32 heads 97 against 91, 700 tokens of 4 heads 24.3 against 22.5; beyond it 900 tokens of 32
    // heads 31.4 against 28.0.
    const double whole = (double)tokens / kC * (packed ? 2.0 / (double)(p.N + 1) : 1.0), split = (double)len / kC * 1.7 + 8;
    if (split > whole) return none;
    return Segments{(int)len, packed ? tokens / len + p.N : segs * p.N};
}

}  // namespace

size_t linear_workspace(const fkda_linear_params& p) {
    const Segments seg = plan(p);
    return seg.len == 0 ? 0 : (size_t)(seg.rows * p.H) * (kD * kD + 1) * sizeof(float);
}

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
    // Single tokens: a fixed batch of them, or a packed batch that must hold some (the host sees only the totals): the step kernel then
    // serves the sequences of at most one token and the chunk kernel the others, whose CTAs find most sequences done.  Step and chunk
    // kernel against the chunk kernel for all, 128 x 1 token, H = 32, fp32 states: 108 us against 303 (as a fixed batch 80); 64 x 1 and
    // 64 x 2: 218 against 304; but nothing but 2 tokens: 328 against 303.  Where one round of SMs walks all chains, a single one that is
    // longer decides: 8 x 1 and 6 tokens, H = 8, 14.1 against 10.8, nothing but single ones 6.1 against 10.5.
    const bool single = p.cu_seqlens == nullptr ? p.T <= 1 : p.T <= p.N || (p.T < 2 * p.N && chains > device_sm_count());
    const bool chunks = p.T > 1;
    a.skip_single = single;
    a.ordered = false;
    a.seg_len = a.seg_rows = 0;
    a.seg_state = a.seg_decay = nullptr;
    a.starve_ms = starve_next();
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
        if (!map4(&maps.q, p.q, p.Hk, p.q_stride) || !map4(&maps.k, p.k, p.Hk, p.k_stride) || !map4(&maps.v, p.v, p.H, p.v_stride) ||
            !map4(&maps.out, p.out, p.H, p.out_stride))
            return FKDA_ERR_LAUNCH;
        const Segments seg = single ? Segments{0, p.N} : plan(p);
        a.seg_len = seg.len;
        a.seg_rows = (int)seg.rows;
        a.seg_state = static_cast<float*>(p.workspace);
        a.seg_decay = a.seg_state + seg.rows * p.H * (kD * kD);
        // The longest first where not all run at once and the last ones are worth what it costs: every CTA ranks all sequences before its
        // first load, 1 us and 0.03 us per sequence.  Ordered against as they come, H = 16: 16 sequences of up to 4 000 tokens 123 us
        // against 156, of up to 1 000 tokens 59 against 67, 32 of these 118 against 117, 64 of these 205 against 195; of up to 60 tokens 16
        // take 27 against 24, 96 168 against 128, and 896 of up to 400 took 5.9 ms against 1.45.  4 to 48 sequences, 1.1 to 4.5 rounds
        // of SMs: 0.74 to 0.97 of the time from 240 tokens per sequence and round on, 0.93 to 1.03 from 160 on, 1.05 to 1.2 below 60.
        const int64_t sms = device_sm_count();
        a.ordered = p.cu_seqlens != nullptr && seg.len == 0 && p.N > 1 && p.N <= kMaxOrdered && chains > sms && p.T >= 160 * p.N * chains / sms;
        // (by the initial state alone: outputs do not depend on whether, and in which type, a final state is asked for)
        const bool exact = a.state_fp32 || p.initial_state == nullptr;
        auto walk = [&](bool states) {
            const int64_t ctas = seg.rows * p.H;
            if (states) return exact ? launch_walk<true, 3>(ctas, stream, a, maps) : launch_walk<true, 2>(ctas, stream, a, maps);
            return exact ? launch_walk<false, 3>(ctas, stream, a, maps) : launch_walk<false, 2>(ctas, stream, a, maps);
        };
        if (seg.len > 0) {
            if (!walk(true) || !launch_dependent(linear_carry_kernel, chains * 16, 256, 0, stream, a)) return FKDA_ERR_LAUNCH;
            launches += 2;
        }
        if (!walk(false)) return FKDA_ERR_LAUNCH;
        ++launches;
    }
    *n_launches = launches;
    return FKDA_OK;
}

int linear_gave_up(cudaStream_t stream, uint32_t* times) { return read_gave_up(stream, times); }

}  // namespace fkda
