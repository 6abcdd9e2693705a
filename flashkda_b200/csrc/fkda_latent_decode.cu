// Latent attention, absorbed form: the queries have been multiplied by the expansion of the keys, so all heads read one vector of
// 576 numbers per token (512 that also serve as the value, 64 rotated ones) straight from a paged cache.  For Tq new tokens
// behind every sequence (rows = new token x head):
//     o_r = sum_j softmax_j(scale q_r . c_j) c_j[0:512],   j < len - Tq + 1 + (new token of r)
//
// The cache is read once: the call is bound by HBM while few rows share a token (1 152 bytes against 2 x 1 088 operations per row)
// and by the tensor cores above some 120 rows.  All tiles of 64 tokens of all sequences form one line that is cut into equal
// pieces, one per CTA, so lengths do not matter to the balance; a sequence that a cut runs through leaves weighted parts that a
// second kernel joins.  A CTA serves 64 rows (groups of CTAs that differ in the rows only walk the same tokens at the same time, so
// the cache tile comes from L2 for all but one).
//
// The 64 x 64 scores are the accumulator Q K^T with one row per lane group of a warp (16 rows per warp); the output is kept transposed,
// 512 dimensions x 64 rows as four accumulators of 128 lanes x 64 columns, so that the cache tile serves as the A operand for the
// value product as it lies (dimension-major), and 256 of the 512 tensor-memory columns are enough.
//
// Numerics: as in the expanded form (fp32 scores, sums and outputs; weights against a reference within 2^8 of the running maximum,
// rounded to bf16 for the value product only); parts are joined in fp32 in the order of the tokens.
#include "fkda_tc5.cuh"

namespace fkda {
namespace {

using namespace tc5;

constexpr int kRows = 64, kTok = 64;         // rows and tokens of a tile
constexpr int kWidth = 576, kValue = 512;
constexpr int kChunks = kWidth / 64;         // 64-dimension tiles of a row or token
constexpr int kChunkBytes = 64 * 128;
constexpr int kStageBytes = kChunks * kChunkBytes;
constexpr int kStages = 2;
constexpr int kThreads = 192;                // softmax warpgroup, a loading and a multiplying warp
constexpr int kMaxSeqs = kStages * kStageBytes / 4;   // tile counts of all sequences pass through the stages' memory
constexpr uint32_t kO = 0, kS = 256;         // tensor-memory columns: four output accumulators, two score buffers

struct DecodeArgs {
    __nv_bfloat16* out;
    float* lse;
    const int32_t *table, *lens;
    float* parts;        // [CTAs][2][kRows][kValue], then their lse [CTAs][2][kRows]
    int64_t out_batch, out_row, table_stride, pages;
    int B, Tq, H, R, row_tiles, groups, page, box, max_pages;
    float scale;
};
struct DecodeMaps {
    CUtensorMap q, cache;
};
struct Bars {
    uint64_t q_full, q_empty, full[kStages], empty[kStages], s_full[2], p_full, o_done, drained;
    uint32_t tmem;
    int abort;
    int first_seq, first_tile, count;
    float factor[kRows];
};
constexpr int kSmem = 1024 + kStageBytes + kStages * kStageBytes + kChunkBytes + 512;
static_assert(sizeof(Bars) <= 512, "barriers");

__device__ __forceinline__ int tiles_of(int len) { return len > 0 ? (len + kTok - 1) / kTok : 0; }
// Length of a sequence as far as its pages go.
__device__ __forceinline__ int length(const DecodeArgs& a, int b) {
    const int x = a.lens[b];
    const int64_t most = (int64_t)a.max_pages * a.page;
    return x < 0 ? 0 : (x > most ? (int)most : x);
}

// The walk of a CTA over its share of the tiles: one sequence's stretch after the other.
struct Walk {
    int b, t, left;
    int len, tiles, until;   // of the current stretch: [t, until)
    __device__ __forceinline__ bool next(const DecodeArgs& a) {
        if (left <= 0) return false;
        len = length(a, b);
        tiles = tiles_of(len);
        while (t >= tiles && b + 1 < a.B) {
            ++b;
            t = 0;
            len = length(a, b);
            tiles = tiles_of(len);
        }
        until = min(tiles, t + left);
        return until > t;
    }
    __device__ __forceinline__ void done() {
        left -= until - t;
        t = until;
    }
};

__global__ void __launch_bounds__(kThreads, 1) latent_decode_kernel(const __grid_constant__ DecodeArgs a, const __grid_constant__ DecodeMaps maps) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* q_smem = smem;                       // [9][64 rows][128 bytes]
    uint8_t* stages = smem + kStageBytes;         // [2][9][64 tokens][128 bytes]
    uint8_t* p_smem = stages + kStages * kStageBytes;
    Bars& bar = *reinterpret_cast<Bars*>(p_smem + kChunkBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(&bar.q_full, 1);
        mbar_init(&bar.q_empty, 1);
        for (int i = 0; i < kStages; ++i) mbar_init(&bar.full[i], 1), mbar_init(&bar.empty[i], 1);
        for (int i = 0; i < 2; ++i) mbar_init(&bar.s_full[i], 1);
        mbar_init(&bar.p_full, 128);
        mbar_init(&bar.o_done, 1);
        mbar_init(&bar.drained, 1);
        bar.abort = 0;
        bar.first_seq = bar.first_tile = bar.count = 0;
        mbar_fence_init();
    }
    if (warp == 5) tmem_alloc(&bar.tmem, 512);
    fence_before();
    grid_dep_launch();
    grid_dep_wait();
    const int rt = (int)(blockIdx.x % a.row_tiles), group = (int)(blockIdx.x / a.row_tiles);
    // ---- where my share begins: tile counts of all sequences, their sum, and the sequence that my first tile is in ----
    int* counts = reinterpret_cast<int*>(stages);
    for (int b = threadIdx.x; b < a.B; b += kThreads) counts[b] = tiles_of(length(a, b));
    __syncthreads();
    fence_after();
    if (warp == 0) {
        int64_t total = 0;
        for (int b = lane; b < a.B; b += 32) total += counts[b];
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
        const int64_t share = (total + a.groups - 1) / a.groups, mine = share * group;
        int64_t seen = 0;
        for (int base = 0; base < a.B && mine < total; base += 32) {
            const int c = base + lane < a.B ? counts[base + lane] : 0;
            int upto = c;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, upto, off);
                if (lane >= off) upto += x;
            }
            const uint32_t behind = __ballot_sync(0xffffffffu, seen + upto > mine);
            if (behind != 0) {
                if (lane == __ffs(behind) - 1) {
                    bar.first_seq = base + lane;
                    bar.first_tile = (int)(mine - (seen + upto - c));
                    bar.count = (int)min(share, total - mine);
                }
                break;
            }
            seen += __shfl_sync(0xffffffffu, upto, 31);
        }
    }
    fence_proxy_async_smem();   // (the stages are written by copies from here on)
    __syncthreads();
    const uint32_t tmem = bar.tmem;
    Walk walk{bar.first_seq, bar.first_tile, bar.count, 0, 0, 0};

    if (warp == 4) {
        // ---- loads ----
        int g = 0, pieces = 0;
        bool ok = true;
        for (; ok && walk.next(a); walk.done(), ++pieces) {
            if (pieces > 0) ok = wait(&bar.q_empty, (pieces - 1) & 1, &bar.abort);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            if (lane == 0) {
                mbar_arrive_expect_tx(&bar.q_full, kStageBytes);
                for (int c = 0; c < kChunks; ++c) tma_load_3d(q_smem + c * kChunkBytes, &maps.q, c * 64, rt * kRows, walk.b, &bar.q_full);
            }
            const int boxes = kTok / a.box;
            for (int t = walk.t; t < walk.until; ++t, ++g) {
                const int stage = g % kStages;
                const int tok = t * kTok + lane * a.box;   // lane = box of the tile
                const bool load = lane < boxes && tok < walk.len;
                int page = 0;
                if (load) {
                    page = a.table[(int64_t)walk.b * a.table_stride + tok / a.page];
                    page = page < 0 || page >= a.pages ? 0 : page;
                }
                if (g >= kStages) ok = wait(&bar.empty[stage], (g / kStages - 1) & 1, &bar.abort);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const int n = __popc(__ballot_sync(0xffffffffu, load));
                if (lane == 0) mbar_arrive_expect_tx(&bar.full[stage], n * a.box * kWidth * 2);
                __syncwarp();
                if (load) {
                    uint8_t* dst = stages + stage * kStageBytes + lane * a.box * 128;
                    for (int c = 0; c < kChunks; ++c) tma_load_3d(dst + c * kChunkBytes, &maps.cache, c * 64, tok % a.page, page, &bar.full[stage]);
                }
                __syncwarp();
            }
            if (!ok) break;
        }
        if (lane == 0) {
            if (pieces > 0) drain(&bar.q_full, (pieces - 1) & 1);
            for (int k = max(0, g - kStages); k < g; ++k) drain(&bar.full[k % kStages], (k / kStages) & 1);
        }
        __syncwarp();
    } else if (warp == 5) {
        // ---- products ----
        if (elect_one()) {
            constexpr uint32_t kIdS = idesc(kRows, kTok, false, false), kIdO = idesc(128, kRows, true, false);
            const uint32_t q_addr = smem_u32(q_smem), st_addr = smem_u32(stages), p_addr = smem_u32(p_smem);
            int g = 0;          // tiles whose scores have been issued
            int done = 0;       // tiles whose value product has been issued
            int piece = 0;
            bool ok = true, prev_first = false;
            auto values = [&](bool first) {   // the value product of tile `done`
                ok = wait(&bar.p_full, done & 1, &bar.abort);
                if (!ok) return;
                fence_after();
                const uint32_t stage = st_addr + (done % kStages) * kStageBytes;
                for (int m = 0; m < 4; ++m)
                    for (int k = 0; k < 4; ++k)
                        mma_ss(tmem + kO + m * kRows, desc(stage + 2 * m * kChunkBytes + k * 2048, kChunkBytes), desc(p_addr + k * 32), kIdO, !first || k > 0);
                commit(&bar.empty[done % kStages]);
                commit(&bar.o_done);
                ++done;
            };
            for (; ok && walk.next(a); walk.done(), ++piece) {
                ok = wait(&bar.q_full, piece & 1, &bar.abort);
                for (int t = walk.t; t < walk.until && ok; ++t) {
                    ok = wait(&bar.full[g % kStages], (g / kStages) & 1, &bar.abort);
                    if (!ok) break;
                    fence_after();
                    const uint32_t stage = st_addr + (g % kStages) * kStageBytes;
                    for (int c = 0; c < kChunks; ++c)
                        for (int k = 0; k < 4; ++k)
                            mma_ss(tmem + kS + (g & 1) * kTok, desc(q_addr + c * kChunkBytes + k * 32), desc(stage + c * kChunkBytes + k * 32), kIdS, (c | k) != 0);
                    commit(&bar.s_full[g & 1]);
                    if (t + 1 == walk.until) commit(&bar.q_empty);
                    if (g > 0) values(prev_first);
                    prev_first = t == walk.t;
                    ++g;
                }
            }
            if (ok && g > 0) values(prev_first);
            commit(&bar.drained);
            drain(&bar.drained, 0);
        }
    } else {
        // ---- weights: warp w has rows 16 w .. 16 w + 15 of the tile, thread 4 g + t columns 8 i + 2 t, + 1 of rows g and g + 8 ----
        const int gr = lane >> 2, tc = lane & 3;
        const int row[2] = {warp * 16 + gr, warp * 16 + gr + 8};
        const uint32_t lanes = (uint32_t)(warp * 32) << 16;
        const float c = a.scale * 1.4426950408889634f, step = 8.0f / c;
        const int news[2] = {(rt * kRows + row[0]) / a.H, (rt * kRows + row[1]) / a.H};   // the rows' new tokens
        int g = 0, piece = 0;
        for (; walk.next(a); walk.done(), ++piece) {
            float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
            const int seen[2] = {min(walk.len, walk.len - a.Tq + 1 + news[0]), min(walk.len, walk.len - a.Tq + 1 + news[1])};
            for (int t = walk.t; t < walk.until; ++t, ++g) {
                wait_warp(&bar.s_full[g & 1], (g >> 1) & 1, &bar.abort);
                fence_after();
                uint32_t s[32];
                ld_frag64(tmem + kS + (g & 1) * kTok + lanes, s);
                wait_ld();
                if ((t + 1) * kTok > walk.len - a.Tq + 1) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (t * kTok + 8 * i + 2 * tc + (k & 1) >= seen[k >> 1]) s[4 * i + k] = 0xff800000u;
                }
                float m[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 32; ++i) m[(i >> 1) & 1] = fmaxf(m[(i >> 1) & 1], f(s[i]));
                bool move[2];
                float factor[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    m[k] = fmaxf(m[k], __shfl_xor_sync(0xffffffffu, m[k], 1));
                    m[k] = fmaxf(m[k], __shfl_xor_sync(0xffffffffu, m[k], 2));
                    move[k] = m[k] > top[k] + step;
                    factor[k] = move[k] ? (top[k] == -INFINITY ? 0.0f : ex2_approx((top[k] - m[k]) * c)) : 1.0f;
                    if (move[k]) top[k] = m[k];
                    sum[k] *= factor[k];
                }
                const bool moved = named_any(1, 128, (move[0] || move[1]) && t > walk.t);
                if (g > 0) {   // the last value product: it has read the weights, and its outputs are there
                    wait_warp(&bar.o_done, (g - 1) & 1, &bar.abort);
                    fence_after();
                }
                if (moved) {
                    if (tc == 0) bar.factor[row[0]] = factor[0], bar.factor[row[1]] = factor[1];
                    named_sync(1, 128);
#pragma unroll 1
                    for (int k = 0; k < 8; ++k) {
                        uint32_t o[32];
                        ld32(tmem + kO + k * 32 + lanes, o);
                        wait_ld();
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] = u(f(o[j]) * bar.factor[(k & 1) * 32 + j]);
                        st32(tmem + kO + k * 32 + lanes, o);
                    }
                    wait_st();
                }
                const float ref[2] = {top[0] == -INFINITY ? 0.0f : -top[0] * c, top[1] == -INFINITY ? 0.0f : -top[1] * c};
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float e0 = ex2_approx(__fmaf_rn(f(s[4 * i + 2 * k]), c, ref[k]));
                        const float e1 = ex2_approx(__fmaf_rn(f(s[4 * i + 2 * k + 1]), c, ref[k]));
                        sum[k] += e0 + e1;
                        *reinterpret_cast<uint32_t*>(p_smem + row[k] * 128 + ((i ^ (row[k] & 7)) << 4) + tc * 4) = pack_bf2(e0, e1);
                    }
                // what lies behind the sequence's last token in the tile is another sequence's, or nobody's
                if ((t + 1) * kTok > walk.len) {
                    const int from = walk.len - t * kTok;
                    uint8_t* stage = stages + (g % kStages) * kStageBytes;
                    const int units = (kTok - from) * 8;
                    for (int k = threadIdx.x; k < units * (kValue / 64); k += 128) {
                        const int ch = k / units;
                        *reinterpret_cast<uint4*>(stage + ch * kChunkBytes + from * 128 + (k - ch * units) * 16) = make_uint4(0, 0, 0, 0);
                    }
                }
                fence_proxy_async_smem();
                fence_before();
                arrive(&bar.p_full);
            }
            // ---- the stretch's outputs: all of the sequence's, or a part with the logarithm of its sum ----
            const bool whole = walk.t == 0 && walk.until == walk.tiles;
            const int slot = ((int)blockIdx.x * 2 + (piece == 0 ? 0 : 1));
            float* part = a.parts + (int64_t)slot * kRows * kValue;
            float* part_lse = a.parts + (int64_t)gridDim.x * 2 * kRows * kValue + (int64_t)slot * kRows;
            named_sync(1, 128);   // (the factors of the last tile have been read)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 1);
                sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 2);
                if (tc == 0) {
                    bar.factor[row[k]] = sum[k] > 0.0f ? 1.0f / sum[k] : (sum[k] == 0.0f ? 0.0f : sum[k]);
                    const float lse = sum[k] == 0.0f ? -INFINITY : (top[k] == -INFINITY ? 0.0f : top[k] * a.scale) + logf(sum[k]);
                    if (!whole) part_lse[row[k]] = lse;
                    else if (a.lse != nullptr && rt * kRows + row[k] < a.R) a.lse[(int64_t)walk.b * a.R + rt * kRows + row[k]] = lse;
                }
            }
            named_sync(1, 128);
            wait_warp(&bar.o_done, (g - 1) & 1, &bar.abort);
            fence_after();
#pragma unroll 1
            for (int k = 0; k < 8; ++k) {
                uint32_t o[32];
                ld32(tmem + kO + k * 32 + lanes, o);
                wait_ld();
                const int dim = (k >> 1) * 128 + warp * 32 + lane, r0 = (k & 1) * 32;
                if (whole) {
                    __nv_bfloat16* dst = a.out + (int64_t)walk.b * a.out_batch + (int64_t)(rt * kRows + r0) * a.out_row + dim;
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (rt * kRows + r0 + j < a.R) dst[j * a.out_row] = f2bf(f(o[j]) * bar.factor[r0 + j]);
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (rt * kRows + r0 + j < a.R) part[(r0 + j) * kValue + dim] = f(o[j]) * bar.factor[r0 + j];
                }
            }
            fence_before();
            named_sync(1, 128);   // (the factors are the next stretch's)
        }
    }
    __syncthreads();
    fence_after();
    if (warp == 5) tmem_dealloc(tmem, 512);
}

// Joins the parts of the sequences that a cut runs through, and writes those without any token.  A CTA: eight rows of a sequence, a
// warp each.
__global__ void __launch_bounds__(256) latent_join_kernel(const __grid_constant__ DecodeArgs a, int ctas) {
    __shared__ int64_t sums[2][8];
    grid_dep_launch();
    grid_dep_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per = (a.R + 7) / 8, b = (int)(blockIdx.x / per), r = (int)(blockIdx.x % per) * 8 + warp;
    int64_t total = 0, before = 0;
    for (int k = threadIdx.x; k < a.B; k += 256) {
        const int n = tiles_of(length(a, k));
        total += n;
        if (k < b) before += n;
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
        total += __shfl_xor_sync(0xffffffffu, total, off);
        before += __shfl_xor_sync(0xffffffffu, before, off);
    }
    if (lane == 0) sums[0][warp] = total, sums[1][warp] = before;
    __syncthreads();
    total = before = 0;
    for (int k = 0; k < 8; ++k) total += sums[0][k], before += sums[1][k];
    if (r >= a.R) return;
    const int n = tiles_of(length(a, b));
    __nv_bfloat16* dst = a.out + (int64_t)b * a.out_batch + (int64_t)r * a.out_row;
    float* lse = a.lse != nullptr ? a.lse + (int64_t)b * a.R + r : nullptr;
    if (n == 0) {
        for (int k = lane; k < kValue / 8; k += 32) *reinterpret_cast<uint4*>(dst + k * 8) = make_uint4(0, 0, 0, 0);
        if (lane == 0 && lse != nullptr) *lse = -INFINITY;
        return;
    }
    const int64_t share = (total + a.groups - 1) / a.groups;
    const int64_t first = before / share, last = (before + n - 1) / share;
    if (first == last) return;
    const int rt = r / kRows, row = r % kRows;
    const float* lses = a.parts + (int64_t)ctas * 2 * kRows * kValue;
    auto slot = [&](int64_t x) { return (x * a.row_tiles + rt) * 2 + (x * share >= before ? 0 : 1); };   // (a CTA's first stretch is its slot 0)
    float top = -INFINITY;
    for (int64_t x = first + lane; x <= last; x += 32) top = fmaxf(top, lses[slot(x) * kRows + row]);
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    const float ref = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f, acc[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) acc[k] = 0.0f;
    for (int64_t x = first; x <= last; ++x) {
        const int64_t s = slot(x);
        const float z = lses[s * kRows + row];
        if (z == -INFINITY) continue;
        const float w = expf(z - ref);
        sum += w;
        const float* src = a.parts + (s * kRows + row) * kValue;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float4 v = *reinterpret_cast<const float4*>(src + k * 128 + lane * 4);
            acc[4 * k] += w * v.x;
            acc[4 * k + 1] += w * v.y;
            acc[4 * k + 2] += w * v.z;
            acc[4 * k + 3] += w * v.w;
        }
    }
    const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
#pragma unroll
    for (int k = 0; k < 4; ++k)
        *reinterpret_cast<uint2*>(dst + k * 128 + lane * 4) =
            make_uint2(pack_bf2(acc[4 * k] * inv, acc[4 * k + 1] * inv), pack_bf2(acc[4 * k + 2] * inv, acc[4 * k + 3] * inv));
    if (lane == 0 && lse != nullptr) *lse = sum == 0.0f ? -INFINITY : ref + logf(sum);
}

int groups_for(int64_t row_tiles) {
    const int sms = device_sm_count();
    return row_tiles >= sms ? 1 : (int)(sms / row_tiles);
}

}  // namespace

size_t latent_decode_workspace(const fkda_latent_decode_params& p) {
    const int64_t row_tiles = (p.Tq * p.H + kRows - 1) / kRows;
    return (size_t)(row_tiles * groups_for(row_tiles)) * 2 * kRows * (kValue + 1) * sizeof(float);
}

int launch_latent_decode(const fkda_latent_decode_params& p, cudaStream_t stream, int* n_launches) {
    if (p.B > kMaxSeqs) return FKDA_ERR_BAD_SHAPE;
    DecodeArgs a;
    a.out = static_cast<__nv_bfloat16*>(p.out);
    a.lse = p.lse;
    a.table = p.block_table;
    a.lens = p.cache_lens;
    a.parts = static_cast<float*>(p.workspace);
    a.out_batch = p.out_stride[0];
    a.out_row = p.out_stride[1];
    a.table_stride = p.block_table_stride;
    a.pages = p.pages;
    a.B = (int)p.B; a.Tq = (int)p.Tq; a.H = (int)p.H; a.R = (int)(p.Tq * p.H);
    a.row_tiles = (a.R + kRows - 1) / kRows;
    a.groups = groups_for(a.row_tiles);
    a.page = (int)p.page_size;
    a.box = p.page_size % 64 == 0 ? 64 : (p.page_size % 32 == 0 ? 32 : 16);
    a.max_pages = (int)p.max_pages;
    a.scale = p.scale;
    DecodeMaps maps;
    const cuuint64_t qdims[3] = {(cuuint64_t)kWidth, (cuuint64_t)a.R, (cuuint64_t)p.B};
    const cuuint64_t qstrides[2] = {(cuuint64_t)p.q_stride[1] * 2, (cuuint64_t)p.q_stride[0] * 2};
    const cuuint32_t qbox[3] = {64u, (cuuint32_t)kRows, 1u};
    const cuuint64_t cdims[3] = {(cuuint64_t)kWidth, (cuuint64_t)p.page_size, (cuuint64_t)(p.pages > 0 ? p.pages : 1)};
    const cuuint64_t cstrides[2] = {(cuuint64_t)p.cache_stride[1] * 2, (cuuint64_t)p.cache_stride[0] * 2};
    const cuuint32_t cbox[3] = {64u, (cuuint32_t)a.box, 1u};
    if (!encode_bf16_map(&maps.q, 3, p.q, qdims, qstrides, qbox) || !encode_bf16_map(&maps.cache, 3, p.cache, cdims, cstrides, cbox))
        return FKDA_ERR_LAUNCH;
    const int ctas = a.row_tiles * a.groups;
    const int64_t joins = p.B * ((a.R + 7) / 8);
    if (joins > 0x7fffffff) return FKDA_ERR_BAD_SHAPE;
    if (!allow_smem<latent_decode_kernel>(kSmem)) return FKDA_ERR_LAUNCH;
    if (!launch_dependent(latent_decode_kernel, ctas, kThreads, kSmem, stream, a, maps)) return FKDA_ERR_LAUNCH;
    if (!launch_dependent(latent_join_kernel, joins, 256, 0, stream, a, ctas)) return FKDA_ERR_LAUNCH;
    *n_launches = 2;
    return FKDA_OK;
}

int decode_gave_up(cudaStream_t stream, int32_t* word) { return read_gave_up(stream, word); }

}  // namespace fkda
