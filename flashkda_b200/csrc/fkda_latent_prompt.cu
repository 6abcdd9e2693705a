// Latent attention, expanded form: every head has keys of its own for the 128 unrotated dimensions and values of its own, and
// shares the 64 rotated ones of the token.  For a prompt:
//     o_i = sum_j softmax_j(scale (q_i[0:128] . k_j + q_i[128:192] . r_j)) v_j
//
// One pass over the keys with the running maximum and sum of the softmax.  A CTA serves 256 rows of one head as two tiles of
// 128, each with a warpgroup of its own that turns scores into weights, one row per thread; while one tile's weights are being made
// the tensor cores work for the other.  Scores and outputs live in tensor memory (2 x 128 + 2 x 128 columns), the weights
// overwrite the scores as the A operand of the product with v.  Keys and values come through eight 16 KB tiles
// (128 tokens x 64 dimensions); the rotated part needs no copy beside the others: it is the third tile of a key block, read
// through a map of its own.  Packed sequences with more keys are taken first.
//
// Measured: 8 192 tokens of 32 heads 595 to 615 us, 0.84 to 0.81 of what cuBLAS sustains, where the power cap holds the clock (passes back
// to back for some tenths of a second); 516 us, 1.33 PFLOP/s, 0.79 of cuBLAS in a burst, in short runs at 1.9 GHz, in which the other
// times below were taken.
// A pair of tiles takes 3 160 cycles per block of keys, for 2 560 of tensor-core work and 2 048 of exponentials; a tile's own
// chain, scores to weights (1 680) to product and the next scores (1 020), with 390 between them, is as long.  One thread's instruction
// stream feeds the tensor cores, so what it has to do beside products counts: barriers per block instead of per 16 KB tile made
// 541 us 520, one product for all 128 dimensions of the values instead of two another 5.  No gain: a quarter of the
// exponentials as polynomials (530 to 539), weights handed over as 96 + 32 keys instead of 64 + 64 (516), scores read in two pieces of 64
// with less code (546 for 541), outputs stored as whole rows by way of shared memory (513 to 516), a persistent form that loads
// the next item's keys beside the last one's outputs (546 to 610).
//
// Numerics: products of bf16 with fp32 sums, weights relative to a reference that follows the running maximum once that is
// 2^8 above it (so weights stay below 2^8 and the sums are exact to 32 bits either way), weights rounded to bf16 for the product
// with v (their relative error, 2^-8 at most, averages out over the keys; the sum and lse use the unrounded weights).
#define FKDA_WAITS_INLINE
#include "fkda_tc5.cuh"

namespace fkda {
namespace {

using namespace tc5;

constexpr int kTile = 128;                   // query rows of a warpgroup, and keys of a block
constexpr int kRows = 2 * kTile;             // query rows of a CTA
constexpr int kSlotBytes = kTile * 128;      // 128 tokens x 64 dimensions
constexpr int kSlots = 8;
constexpr int kKeyTiles = 3, kValueTiles = 2;
// Where block i's tiles lie: the keys' first two in one of three pairs of slots, where block i - 3's lay, block i - 2's values after
// them; its values in the pair of block i - 1's keys; the keys' third tile in one of two more slots.  So the tiles of the values are
// always neighbours (one product covers their 128 dimensions), and a block's keys wait for nothing younger than block i - 2.
__device__ __forceinline__ int key_slot(int i, int c) { return c < 2 ? 2 * (i % 3) + c : 6 + (i & 1); }
__device__ __forceinline__ int value_slot(int i) { return 2 * ((i + 2) % 3); }
constexpr int kThreads = 384;                // two softmax warpgroups, and one with a loading and a multiplying warp
// Registers of a thread: 168 at launch, then 208 for a row's 128 scores and what is made of them; 2 x 208 + 88 = 3 x 168
constexpr int kRegsRow = 208, kRegsRest = 88;
static_assert(2 * kRegsRow + kRegsRest <= 3 * 168, "a block has no more");
constexpr uint32_t kS = 0, kO = 256;         // tensor-memory columns: scores (and weights) of the two tiles, outputs

struct PromptMaps {
    CUtensorMap q, k, r, v;
};
struct PromptArgs {
    __nv_bfloat16* out;
    float* lse;
    const int64_t *cu_q, *cu_k;
    int64_t T, Tk, N, out_batch, out_token, out_head;
    int H;
    bool ordered;          // packed sequences: those with more keys first
    float scale;
    int causal;
    int starve_ms;         // test hook: nothing is loaded, and a wait gives up after so long
};

constexpr int kMaxOrdered = 32;              // packed sequences that are taken in the order of their keys
struct Bars {
    // (keys and values of block i: the barriers i & 1)
    uint64_t q_full[2], k_full[2], v_full[2], k_empty[2], v_empty[2], s_full[2], p_full[2][2], o_done[2], drained;
    uint32_t tmem;
    int abort;
    int order[kMaxOrdered];
};

constexpr int kSmem = (2 * kKeyTiles + kSlots) * kSlotBytes + ((int)sizeof(Bars) + 127) / 128 * 128;
static_assert(kSmem <= 232448, "shared memory of an SM");

// Where a CTA's rows are: sequence, first row, and the extents of queries and keys.
struct Place {
    int64_t q0, k0, b;     // first token of the sequence's queries and keys, batch row
    int len_q, len_k, row0;
    bool any;
};
// `order`: the sequences with more keys first, so that a long one does not start when the others are done; or null, as they come.
__device__ __forceinline__ Place locate(const PromptArgs& a, const int* order, int64_t slot, int lane) {
    Place p;
    if (a.cu_q == nullptr) {
        // long rows first: the last block of every sequence, then the one in front of it, ...
        const int64_t tiles = (a.T + kRows - 1) / kRows, t = slot / a.N;
        p.b = slot - t * a.N;
        p.q0 = p.k0 = 0;
        p.len_q = (int)a.T;
        p.len_k = (int)a.Tk;
        p.row0 = (int)(tiles - 1 - t) * kRows;
        p.any = true;
        return p;
    }
    int64_t seen = 0;
    p.any = false;
    p.b = 0;
    for (int64_t base = 0; base < a.N; base += 32) {
        int64_t n = base + lane, lo = 0, len = 0;
        if (n < a.N) {
            if (order != nullptr) n = order[n];
            lo = a.cu_q[n] < 0 ? 0 : a.cu_q[n];
            const int64_t hi = a.cu_q[n + 1] > a.T ? a.T : a.cu_q[n + 1];
            len = hi > lo ? hi - lo : 0;
        }
        const int tiles = (int)((len + kRows - 1) / kRows);
        int upto = tiles;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, upto, off);
            if (lane >= off) upto += x;
        }
        const uint32_t behind = __ballot_sync(0xffffffffu, seen + upto > slot);
        if (behind != 0) {
            const int src = __ffs(behind) - 1;
            const int64_t first = seen + __shfl_sync(0xffffffffu, upto - tiles, src);
            const int64_t seq = __shfl_sync(0xffffffffu, n, src);
            p.q0 = __shfl_sync(0xffffffffu, lo, src);
            p.len_q = (int)__shfl_sync(0xffffffffu, len, src);
            p.row0 = (int)((p.len_q + kRows - 1) / kRows - 1 - (slot - first)) * kRows;
            const int64_t klo = a.cu_k[seq] < 0 ? 0 : a.cu_k[seq], khi = a.cu_k[seq + 1] > a.Tk ? a.Tk : a.cu_k[seq + 1];
            p.k0 = klo;
            p.len_k = khi > klo ? (int)(khi - klo) : 0;
            p.any = true;
            return p;
        }
        seen += __shfl_sync(0xffffffffu, upto, 31);
    }
    return p;
}

// (Not inlined: inlined it made 960 us of 546 for 8 192 tokens of 32 heads; probably the compiler no longer knows then that the warps
// are converged.)
__device__ __noinline__ void make_order(const PromptArgs& a, int* lens, int* order) {
    for (int i = threadIdx.x; i < a.N; i += kThreads) lens[i] = (int)(a.cu_k[i + 1] - a.cu_k[i]);
    fence_proxy_async_smem();
    __syncthreads();
    for (int i = threadIdx.x; i < a.N; i += kThreads) {
        const int len = lens[i];
        int rank = 0;
#pragma unroll 1
        for (int j = 0; j < (int)a.N; ++j) rank += lens[j] > len || (lens[j] == len && j < i) ? 1 : 0;
        order[rank] = i;
    }
    fence_proxy_async_smem();
    __syncthreads();
}

__global__ void __launch_bounds__(kThreads, 1) latent_prompt_kernel(const __grid_constant__ PromptArgs a, const __grid_constant__ PromptMaps maps) {
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* q_smem = smem;                                        // [2 tiles][3][128 rows][128 bytes]
    uint8_t* ring = smem + 2 * kKeyTiles * kSlotBytes;
    Bars& bar = *reinterpret_cast<Bars*>(ring + kSlots * kSlotBytes);
    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(&bar.q_full[0], 1), mbar_init(&bar.q_full[1], 1);
        for (int i = 0; i < 2; ++i) mbar_init(&bar.k_full[i], 1), mbar_init(&bar.v_full[i], 1), mbar_init(&bar.k_empty[i], 1), mbar_init(&bar.v_empty[i], 1);
        for (int i = 0; i < 2; ++i) mbar_init(&bar.s_full[i], 1), mbar_init(&bar.p_full[i][0], kTile), mbar_init(&bar.p_full[i][1], kTile), mbar_init(&bar.o_done[i], 1);
        mbar_init(&bar.drained, 1);
        bar.abort = 0;
        mbar_fence_init();
    }
    if (warp == 9) tmem_alloc(&bar.tmem, 512);
    fence_before();
    grid_dep_launch();
    grid_dep_wait();
    __syncthreads();
    fence_after();
    constexpr uint32_t tmem = 0;   // (all columns are this CTA's)
    const int* order = nullptr;
    if (a.ordered) {
        make_order(a, reinterpret_cast<int*>(ring), bar.order);
        order = bar.order;
    }
    Place p = locate(a, order, blockIdx.x / a.H, lane);
    p.any = p.any && as_assumed(smem, bar.tmem);
    const int h = (int)(blockIdx.x % (uint32_t)a.H);
    // key blocks of the two tiles: a row sees the keys up to its own place counted from the ends
    int n[2] = {0, 0};
    if (p.any) {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const int last = min(p.row0 + (w + 1) * kTile, p.len_q);   // one past the tile's last row
            const int seen = a.causal ? min(p.len_k, max(0, p.len_k - p.len_q + last)) : p.len_k;
            n[w] = uniform(p.row0 + w * kTile < p.len_q ? (seen + kTile - 1) / kTile : 0);
        }
    }
    const int blocks = max(n[0], n[1]);

    if (warp >= 8) {
    regs_dec<kRegsRest>();
    if (warp == 8) {
        // ---- loads: the queries, then for every block its keys (two tiles of the head's, one of the token's) and values ----
        if (a.starve_ms > 0) {
            starve(&bar.k_full[0], a.starve_ms, &bar.abort);
        } else if (blocks > 0) {
            const uint32_t q_addr = smem_u32(q_smem), ring_addr = smem_u32(ring), leader = elect_one();
            const int q0 = uniform((int)(p.q0 + p.row0)), row = uniform((int)p.b), k0 = uniform((int)p.k0);
            int keys = 0, values = 0;   // blocks of either that have been asked for
            auto empty = [&](uint64_t* b, int phase) { return __all_sync(0xffffffffu, wait_free(b, phase & 1, &bar.abort)) != 0; };
            auto slot = [&](int s) { return ring_addr + s * kSlotBytes; };
#pragma unroll 1
            for (int i = 0; i < blocks; ++i) {
                const int t = k0 + i * kTile;
                if (i >= 2 && !empty(&bar.v_empty[i & 1], (i >> 1) - 1)) break;   // (the keys of block i - 2 were waited for below)
                uint64_t* full = &bar.k_full[i & 1];
                expect(full, kKeyTiles * kSlotBytes, leader);
                load_4d(slot(key_slot(i, 0)), &maps.k, 0, h, t, row, full, leader);
                load_4d(slot(key_slot(i, 1)), &maps.k, 64, h, t, row, full, leader);
                load_3d(slot(key_slot(i, 2)), &maps.r, 0, t, row, full, leader);
                ++keys;
                if (i == 0) {
#pragma unroll 1
                    for (int w = 0; w < 2; ++w) {
                        expect(&bar.q_full[w], kKeyTiles * kSlotBytes, leader);
#pragma unroll
                        for (int c = 0; c < kKeyTiles; ++c) load_4d(q_addr + (w * kKeyTiles + c) * kSlotBytes, &maps.q, c * 64, h, q0 + w * kTile, row, &bar.q_full[w], leader);
                    }
                }
                if (i >= 1 && !empty(&bar.k_empty[(i - 1) & 1], (i - 1) >> 1)) break;
                full = &bar.v_full[i & 1];
                expect(full, kValueTiles * kSlotBytes, leader);
                load_4d(slot(value_slot(i)), &maps.v, 0, h, t, row, full, leader);
                load_4d(slot(value_slot(i) + 1), &maps.v, 64, h, t, row, full, leader);
                ++values;
            }
            drain(&bar.q_full[0], 0);
            drain(&bar.q_full[1], 0);
#pragma unroll 1
            for (int i = max(0, keys - 2); i < keys; ++i) drain(&bar.k_full[i & 1], (i >> 1) & 1);
#pragma unroll 1
            for (int i = max(0, values - 2); i < values; ++i) drain(&bar.v_full[i & 1], (i >> 1) & 1);
            __syncwarp();
        }
    } else if (warp == 9) {
        // ---- products ----
        if (blocks > 0) {
            constexpr uint32_t kIdS = idesc(kTile, kTile, false, false), kIdO = idesc(kTile, 128, false, true);
            const uint32_t q_desc = desc(smem_u32(q_smem)), k_desc0 = desc(smem_u32(ring)), v_desc0 = desc(smem_u32(ring), kSlotBytes), leader = elect_one();
            auto scores = [&](int w, int i, bool first) {   // tile w against key block i
#pragma unroll
                for (int c = 0; c < kKeyTiles; ++c) {
                    if (first && c == 0) wait_warp(&bar.k_full[i & 1], (i >> 1) & 1, &bar.abort);
                    if (c == 0) fence_after();
                    const uint32_t k_desc = k_desc0 + key_slot(i, c) * (kSlotBytes / 16);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma_ss(tmem + kS + w * kTile, q_desc + ((w * kKeyTiles + c) * kSlotBytes + k * 32) / 16, k_desc + k * 32 / 16, kIdS, (c | k) != 0, leader);
                }
                commit(&bar.s_full[w], leader);
            };
#pragma unroll
            for (int w = 0; w < 2; ++w)
                if (n[w] > 0) {
                    wait_warp(&bar.q_full[w], 0, &bar.abort);
                    scores(w, 0, w == 0 || n[0] == 0);
                }
            commit(&bar.k_empty[0], leader);
#pragma unroll 1
            for (int i = 0; i < blocks; ++i) {
                const int first_v = i < n[0] ? 0 : 1, last_v = i < n[1] ? 1 : 0;
                const int first_k = i + 1 < n[0] ? 0 : 1, last_k = i + 1 < n[1] ? 1 : 0;
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    if (i >= n[w]) continue;
#pragma unroll
                    for (int half = 0; half < 2; ++half) {   // 64 keys
                        wait_warp(&bar.p_full[w][half], i & 1, &bar.abort);
                        if (half == 0 && w == first_v) wait_warp(&bar.v_full[i & 1], (i >> 1) & 1, &bar.abort);
                        fence_after();
                        const uint32_t v_desc = v_desc0 + value_slot(i) * (kSlotBytes / 16);
#pragma unroll
                        for (int k = 4 * half; k < 4 * half + 4; ++k)
                            mma_ts(tmem + kO + w * kTile, tmem + kS + w * kTile + k * 8, v_desc + k * 2048 / 16, kIdO, i > 0 || k > 0, leader);
                    }
                    commit(&bar.o_done[w], leader);
                    if (w == last_v) commit(&bar.v_empty[i & 1], leader);
                    if (i + 1 < n[w]) {
                        scores(w, i + 1, w == first_k);
                        if (w == last_k) commit(&bar.k_empty[(i + 1) & 1], leader);
                    }
                }
            }
            commit(&bar.drained, leader);
            drain(&bar.drained, 0);
        }
    }
    } else {
        // ---- weights: thread = row ----
        regs_inc<kRegsRow>();
        const int w = warp >> 2, n0 = n[0], blocks_w = w == 0 ? n[0] : n[1];
        const int row = p.row0 + w * kTile + (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + kS + w * kTile + lanes, to = tmem + kO + w * kTile + lanes;
        const float c = a.scale * 1.4426950408889634f;
        int seen = p.any ? (a.causal ? p.len_k - p.len_q + row + 1 : p.len_k) : 0;
        seen = min(max(seen, 0), p.any ? p.len_k : 0);
        const int least = p.any ? (a.causal ? p.len_k - p.len_q + p.row0 + w * kTile + 1 : p.len_k) : 0;   // what the tile's first row sees
        const float step = 8.0f / c;
        float top = -INFINITY, sum = 0.0f;
#pragma unroll 1
        for (int i = 0; i < blocks_w; ++i) {
            uint32_t s[128];
            if (i > 0) wait_warp(&bar.o_done[w], (i - 1) & 1, &bar.abort);   // (issued in front of these scores)
            wait_warp(&bar.s_full[w], i & 1, &bar.abort);
            fence_after();
#pragma unroll
            for (int k = 0; k < 4; ++k) ld32(ts + k * 32, s + k * 32);
            wait_ld();
            if ((i + 1) * kTile > least || (i + 1) * kTile > p.len_k) {
#pragma unroll
                for (int k = 0; k < 128; ++k) s[k] = i * kTile + k < seen ? s[k] : 0xff800000u;
            }
            float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int k = 0; k < 128; k += 2) most[(k >> 1) & 3] = fmaxf(fmaxf(f(s[k]), f(s[k + 1])), most[(k >> 1) & 3]);
            const float m = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
            // the reference moves where the maximum is 2^8 above it; then what was summed so far is scaled down
            const bool move = m > top + step || (top == -INFINITY && m > -INFINITY);
            if (__any_sync(0xffffffffu, move)) {
                const float factor = move ? (top == -INFINITY ? 0.0f : ex2_approx((top - m) * c)) : 1.0f;
                if (move) top = m;
                sum *= factor;
                if (i > 0) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t o[32];
                        ld32(to + k * 32, o);
                        wait_ld();
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] = u(f(o[j]) * factor);
                        st32(to + k * 32, o);
                    }
                }
            }
            const float ref = top == -INFINITY ? 0.0f : -top * c;
            // values behind the sequence's last key are another sequence's, or nobody's: nothing times them must be nothing
            if ((i + 1) * kTile > p.len_k && w == (i < n0 ? 0 : 1)) {
                const int from = p.len_k - i * kTile;
                wait_warp(&bar.v_full[i & 1], (i >> 1) & 1, &bar.abort);
                for (int v = 0; v < kValueTiles; ++v) {
                    uint4* dst = reinterpret_cast<uint4*>(ring + (value_slot(i) + v) * kSlotBytes);
                    for (int k = from * 8 + (threadIdx.x & 127); k < kTile * 8; k += 128) dst[k] = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async_smem();
            }
            float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int half = 0; half < 2; ++half) {   // the product with the values starts on the first 64 keys
                uint32_t* x = s + half * 64;
#pragma unroll
                for (int k = 0; k < 64; k += 2) {
                    fma2(x[k], x[k + 1], c, ref);
                    x[k] = u(ex2_approx(f(x[k])));
                    x[k + 1] = u(ex2_approx(f(x[k + 1])));
                    add2(part[k & 2], part[(k & 2) + 1], x[k], x[k + 1]);
                    x[k >> 1] = pack_bf2(f(x[k]), f(x[k + 1]));
                }
                st32(ts + half * 32, x);
                wait_st();
                fence_before();
                arrive(&bar.p_full[w][half]);
            }
            sum += (part[0] + part[1]) + (part[2] + part[3]);
        }
        if (blocks_w > 0) {
            wait_warp(&bar.o_done[w], (blocks_w - 1) & 1, &bar.abort);
            fence_after();
        }
        const bool mine = p.any && row < p.len_q;
        const int64_t tok = p.q0 + row;
        const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);   // (a sum that is not a number stays one)
        __nv_bfloat16* dst = a.out + p.b * a.out_batch + tok * a.out_token + h * a.out_head;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            uint32_t o[32];
            if (blocks_w > 0) {
                ld32(to + k * 32, o);
                wait_ld();
            } else {
#pragma unroll
                for (int j = 0; j < 32; ++j) o[j] = 0u;
            }
            if (mine) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint4 x;
                    x.x = pack_bf2(f(o[8 * j]) * inv, f(o[8 * j + 1]) * inv);
                    x.y = pack_bf2(f(o[8 * j + 2]) * inv, f(o[8 * j + 3]) * inv);
                    x.z = pack_bf2(f(o[8 * j + 4]) * inv, f(o[8 * j + 5]) * inv);
                    x.w = pack_bf2(f(o[8 * j + 6]) * inv, f(o[8 * j + 7]) * inv);
                    *reinterpret_cast<uint4*>(dst + k * 32 + j * 8) = x;
                }
            }
        }
        if (mine && a.lse != nullptr)
            a.lse[(p.b * a.T + tok) * a.H + h] = sum == 0.0f ? -INFINITY : (top == -INFINITY ? 0.0f : top * a.scale) + logf(sum);
        fence_before();
    }
    __syncthreads();
    fence_after();
    if (warp == 9) tmem_dealloc(tmem, 512);
}

}  // namespace

int launch_latent_prompt(const fkda_latent_params& p, cudaStream_t stream, int* n_launches) {
    PromptMaps maps;
    auto map4 = [](CUtensorMap* m, const void* base, int64_t d, int64_t h, int64_t t, int64_t b, const int64_t* st) {
        const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)h, (cuuint64_t)t, (cuuint64_t)b};
        const cuuint64_t strides[3] = {(cuuint64_t)st[2] * 2, (cuuint64_t)st[1] * 2, (cuuint64_t)st[0] * 2};
        const cuuint32_t box[4] = {64u, 1u, (cuuint32_t)kTile, 1u};
        return encode_bf16_map(m, 4, base, dims, strides, box);
    };
    const cuuint64_t rdims[3] = {64u, (cuuint64_t)p.Tk, (cuuint64_t)p.B};
    const cuuint64_t rstrides[2] = {(cuuint64_t)p.k_rope_stride[1] * 2, (cuuint64_t)p.k_rope_stride[0] * 2};
    const cuuint32_t rbox[3] = {64u, (cuuint32_t)kTile, 1u};
    if (p.Tk > 0) {
        if (!map4(&maps.k, p.k, 128, p.H, p.Tk, p.B, p.k_stride) || !map4(&maps.v, p.v, 128, p.H, p.Tk, p.B, p.v_stride) ||
            !encode_bf16_map(&maps.r, 3, p.k_rope, rdims, rstrides, rbox))
            return FKDA_ERR_LAUNCH;
    }
    if (!map4(&maps.q, p.q, 192, p.H, p.T, p.B, p.q_stride)) return FKDA_ERR_LAUNCH;
    if (p.Tk == 0) maps.k = maps.v = maps.r = maps.q;   // (no key is read)
    PromptArgs a;
    a.out = static_cast<__nv_bfloat16*>(p.out);
    a.lse = p.lse;
    a.cu_q = p.cu_seqlens;
    a.cu_k = p.cu_seqlens_k;
    a.T = p.T; a.Tk = p.Tk; a.N = p.N;
    a.out_batch = p.out_stride[0]; a.out_token = p.out_stride[1]; a.out_head = p.out_stride[2];
    a.H = (int)p.H;
    a.scale = p.scale;
    a.causal = p.causal;
    a.starve_ms = starve_next();
    const int64_t tiles = (p.T + kRows - 1) / kRows;
    const int64_t ctas = (p.cu_seqlens != nullptr ? p.T / kRows + p.N : tiles * p.B) * p.H;   // (ragged: never fewer than there are)
    if (ctas > 0x7fffffff) return FKDA_ERR_BAD_SHAPE;
    // The sequences with more keys first where a few rounds of SMs serve some sequences of some length: every CTA ranks all of them before
    // its first load.  Ordered against as they come, H = 8: 8 sequences of up to 1 000 tokens 29.6 us against 31.9, of up to 4 000 131
    // against 139, 24 of up to 1 000 62.6 against 64.0; but 12 of up to 4 000 (six rounds) 197 against 193, 24 of up to 100 16.5 against
    // 14.4, and 512 of up to 40 took 1 180 against 250.
    const int64_t sms = device_sm_count();
    a.ordered = p.cu_seqlens != nullptr && p.N >= 8 && p.N <= kMaxOrdered && p.T >= 256 * p.N && ctas > sms && ctas <= 4 * sms;
    if (!allow_smem<latent_prompt_kernel>(kSmem)) return FKDA_ERR_LAUNCH;
    if (!launch_dependent(latent_prompt_kernel, ctas, kThreads, kSmem, stream, a, maps)) return FKDA_ERR_LAUNCH;
    *n_launches = 1;
    return FKDA_OK;
}

int prompt_gave_up(cudaStream_t stream, uint32_t* times) { return read_gave_up(stream, times); }

}  // namespace fkda
