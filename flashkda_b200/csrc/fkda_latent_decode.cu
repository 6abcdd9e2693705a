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
// Measured: a tile of 64 tokens takes a CTA some 2 300 cycles of products (36 of 64 x 64 at 42, 16 of 128 x 64 at 49) and 1 100 of weights,
// which run beside the next tile's scores, against 3 100 for its bytes, and yet some 4 500 in all: neither HBM (59 % of its peak) nor the tensor
// cores (46 %) bound the walk.  148 sequences of 4 096 tokens of 64 heads 148 us, 0.72 of the copy bandwidth; 64 of 4 000, most of them cut,
// 89 to 98 (0.51 to 0.46); 128 uneven ones up to 8 192 165 to 174 in passes back to back, 153 in short runs (0.59 to 0.56, 0.64).  384 rows
// per token: 335 to 342 us, 321 in short runs, 0.40 of cuBLAS.  One sequence of 2 989 tokens: 14 us, of which 6.5 are the walk.
//
// Numerics: as in the expanded form (fp32 scores, sums and outputs; weights against a reference within 2^8 of the running maximum,
// rounded to bf16 for the value product only); parts are joined in fp32 in the order of the tokens.
#include <algorithm>
#include <type_traits>

#define FKDA_WAITS_INLINE
#include "fkda_tc5.cuh"

namespace fkda {
namespace {

using namespace tc5;

constexpr int kRows = 64, kTok = 64;         // rows and tokens of a tile
constexpr int kWidth = 576, kValue = 512;
constexpr int kChunks = kWidth / 64;         // 64-dimension tiles of a row or token
constexpr int kChunkBytes = 64 * 128;
constexpr int kStageBytes = kChunks * kChunkBytes;
constexpr int kStages = 2;                   // (tile g's is g & 1)
constexpr int kGroups = 5;                   // of a stage, loaded and freed apart: four pairs of 64-dimension tiles, and the rotated one
constexpr int kThreads = 256;                // softmax warpgroup, three loading warps (4, 6, 7) and a multiplying one (5)
constexpr int kLoaders = 3;
constexpr int kMaxSeqs = kStages * kStageBytes / 4;   // tile counts of all sequences pass through the stages' memory
constexpr uint32_t kO = 0, kS = 256;         // tensor-memory columns: four output accumulators, two score buffers

struct DecodeArgs {
    __nv_bfloat16* out;
    float* lse;
    const int32_t *table, *lens;
    const __nv_bfloat16* cache;
    int64_t page_stride;     // elements from page to page where a page's tokens lie one behind the other, else 0 (no fetching ahead)
    float* parts;        // [CTAs][2][kRows][kValue], then their lse [CTAs][2][kRows]
    int4* spans;         // [B] first and last group of CTAs with tiles of a sequence, whether the first begins with it
    int64_t out_batch, out_row, table_stride, pages;
    int B, Tq, H, R, row_tiles, groups, page, box, max_pages;
    float scale;
    int starve_ms;       // test hook: nothing is loaded, and a wait gives up after so long
};
struct DecodeMaps {
    CUtensorMap q, cache;
};
struct Bars {
    uint64_t q_full, q_empty, full[kStages][kGroups], empty[kStages][kGroups], s_full[2], p_full, o_done, drained;
    uint32_t tmem;
    int abort;
    int first_seq, first_tile, count;
    alignas(16) float factor[kRows];
};
constexpr int kSmem = kStageBytes + kStages * kStageBytes + kChunkBytes + 640;
static_assert(sizeof(Bars) <= 640 && kSmem <= 232448, "shared memory of an SM");

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
    // (Not inlined: inlined, such a loop made the products slower, as it did in the prompts' kernel.)
    __device__ __noinline__ bool next(const DecodeArgs& a) {
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
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* q_smem = smem;                       // [9][64 rows][128 bytes]
    uint8_t* stages = smem + kStageBytes;         // [2][9][64 tokens][128 bytes]
    uint8_t* p_smem = stages + kStages * kStageBytes;
    Bars& bar = *reinterpret_cast<Bars*>(p_smem + kChunkBytes);
    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(&bar.q_full, 1);
        mbar_init(&bar.q_empty, 1);
        for (int i = 0; i < kStages; ++i)
            for (int j = 0; j < kGroups; ++j) mbar_init(&bar.full[i][j], 1), mbar_init(&bar.empty[i][j], 1);
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
        for (int base = 0, turn = 0; base < a.B; base += 32, turn = turn + 1 == a.groups ? 0 : turn + 1) {
            const int c = base + lane < a.B ? counts[base + lane] : 0;
            int upto = c;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, upto, off);
                if (lane >= off) upto += x;
            }
            const int64_t before = seen + upto - c;
            if (mine < total && before <= mine && mine < before + c) {
                bar.first_seq = base + lane;
                bar.first_tile = (int)(mine - before);
                bar.count = (int)min(share, total - mine);
            }
            if (rt == 0 && turn == group && base + lane < a.B) {   // (the groups note 32 sequences each in turn)
                const int first = c > 0 ? (int)(before / share) : 0, last = c > 0 ? (int)((before + c - 1) / share) : 0;
                a.spans[base + lane] = make_int4(first, last, first * share == before ? 1 : 0, 0);
            }
            seen += __shfl_sync(0xffffffffu, upto, 31);
        }
    } else if (warp < 4) {
        // sequences without any token: nothing
        for (int b = group; b < a.B; b += a.groups) {
            if (counts[b] != 0) continue;
            for (int i = threadIdx.x - 32; i < kRows * (kValue / 8); i += 96) {
                const int row = rt * kRows + i / (kValue / 8);
                if (row >= a.R) break;
                *reinterpret_cast<uint4*>(a.out + (int64_t)b * a.out_batch + (int64_t)row * a.out_row + i % (kValue / 8) * 8) = make_uint4(0, 0, 0, 0);
                if (i % (kValue / 8) == 0 && a.lse != nullptr) a.lse[(int64_t)b * a.R + row] = -INFINITY;
            }
        }
    }
    fence_proxy_async_smem();   // (the stages are written by copies from here on)
    __syncthreads();
    constexpr uint32_t tmem = 0;   // (all columns are this CTA's)
    Walk walk{(int)uniform(bar.first_seq), (int)uniform(bar.first_tile), (int)uniform(as_assumed(smem, bar.tmem) ? bar.count : 0), 0, 0, 0};

    if (warp == 4 || warp > 5) {
        // ---- loads: a tile in groups of its dimensions, box by box (pages may end inside it); two tiles on are fetched into L2, so that a
        //      stage that was freed is full again without waiting for HBM.  A copy takes some 120 cycles to issue, and pages of 16 tokens make
        //      36 of them per tile: three warps share the groups ----
        const int who = warp == 4 ? 0 : warp - 5;
        const uint32_t q_addr = smem_u32(q_smem), st_addr = smem_u32(stages), leader = elect_one();
        const int boxes = kTok / a.box;
        int g = 0, pieces = 0, asked = 0, issued[2] = {0, 0};   // (tiles of my first and second group)
        bool ok = true;
        if (a.starve_ms > 0) starve(&bar.full[0][who], a.starve_ms, &bar.abort), ok = false;
        auto page_of = [&](int tok) {
            const int page = a.table[(int64_t)walk.b * a.table_stride + tok / a.page];
            return page < 0 || page >= a.pages ? 0 : page;
        };
        auto fetch_ahead = [&](int t) {   // lane = box of the tile
            const int tok = t * kTok + lane * a.box;
            if (a.page_stride == 0 || t >= walk.until || lane >= boxes || tok >= walk.len) return;
            const __nv_bfloat16* from = a.cache + (int64_t)page_of(tok) * a.page_stride + (int64_t)(tok % a.page) * kWidth;
            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(from), "r"(a.box * kWidth * 2) : "memory");
        };
#pragma unroll 1
        for (; ok && walk.next(a); walk.done(), ++pieces) {
            if (who == 2) fetch_ahead(walk.t + 1);
            __syncwarp();
#pragma unroll 1
            for (int t = walk.t; t < walk.until; ++t, ++g) {
                const int tok = t * kTok + lane * a.box;
                const bool load = lane < boxes && tok < walk.len;
                const int my_page = load ? page_of(tok) : 0, my_row = load ? tok % a.page : 0, n = __popc(__ballot_sync(0xffffffffu, load));
                if (who == 2) fetch_ahead(t + 2);
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int j = who + i * kLoaders;
                    if (j >= kGroups) break;
                    if (g >= kStages) ok = __all_sync(0xffffffffu, wait(&bar.empty[g & 1][j], ((g >> 1) - 1) & 1, &bar.abort));
                    if (!ok) break;
                    const int width = j == kGroups - 1 ? 1 : 2;
                    uint64_t* full = &bar.full[g & 1][j];
                    expect(full, n * a.box * 128 * width, leader);
#pragma unroll 1
                    for (int b = 0; b < n; ++b) {
                        const int page = __shfl_sync(0xffffffffu, my_page, b), row = __shfl_sync(0xffffffffu, my_row, b);
                        const uint32_t dst = st_addr + (g & 1) * kStageBytes + 2 * j * kChunkBytes + b * a.box * 128;
                        load_3d(dst, &maps.cache, j * 128, row, page, full, leader);
                        if (width == 2) load_3d(dst + kChunkBytes, &maps.cache, j * 128 + 64, row, page, full, leader);
                    }
                    issued[i] = g + 1;
                }
                if (!ok) break;
                if (t > walk.t || who != 0) continue;
                // the stretch's queries, once the last one's have been read
                if (pieces > 0) ok = __all_sync(0xffffffffu, wait(&bar.q_empty, (pieces - 1) & 1, &bar.abort));
                if (!ok) break;
                expect(&bar.q_full, kStageBytes, leader);
                ++asked;
                const int seq = uniform(walk.b);
#pragma unroll 1
                for (int c = 0; c < kChunks; ++c) load_3d(q_addr + c * kChunkBytes, &maps.q, c * 64, rt * kRows, seq, &bar.q_full, leader);
            }
            if (!ok) break;
        }
        if (asked > 0) drain(&bar.q_full, (asked - 1) & 1);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            for (int k = max(0, issued[i] - kStages); k < issued[i]; ++k) drain(&bar.full[k & 1][who + i * kLoaders], (k >> 1) & 1);
        __syncwarp();
    } else if (warp == 5) {
        // ---- products: two lines of work, each taken up as soon as what it waits for is there: the scores of tile `g`, group by group of its
        //      dimensions, at most one tile ahead of the value product of tile `done`.  (It never multiplies, and so never frees, what has not
        //      landed: the loads need no look at the abort flag.) ----
        const uint32_t q_desc = desc(smem_u32(q_smem)), k_desc = desc(smem_u32(stages)), leader = elect_one();
        const uint32_t v_desc = desc(smem_u32(stages), kChunkBytes), p_desc = desc(smem_u32(p_smem));
        // the groups that are there, from the next one on (stage and group in the code, so that the operands are constants)
        auto scores = [q_desc, k_desc, leader](auto stage, uint32_t there, int& group) {
            constexpr int kStage = decltype(stage)::value;
#pragma unroll
            for (int j = 0; j < kGroups; ++j) {
                if (group != j || (there >> j & 1) == 0) continue;
#pragma unroll
                for (int i = 8 * j; i < min(8 * j + 8, 4 * kChunks); ++i) {
                    const int at = (i / 4 * kChunkBytes + i % 4 * 32) / 16;
                    mma_ss(kS + kStage * kTok, q_desc + at, k_desc + kStage * (kStageBytes / 16) + at, idesc(kRows, kTok, false, false), i != 0, leader);
                }
                ++group;
            }
        };
        auto values = [v_desc, p_desc, leader, &bar](auto stage, uint32_t adds) {
            constexpr int kStage = decltype(stage)::value;
#pragma unroll
            for (int m = 0; m < 4; ++m) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    mma_ss(kO + m * kRows, v_desc + (kStage * kStageBytes + 2 * m * kChunkBytes + k * 2048) / 16, p_desc + k * 32 / 16, idesc(128, kRows, true, false), k > 0 ? 1 : adds, leader);
                commit(&bar.empty[kStage][m], leader);
            }
        };
        int g = 0, group_of = 0, done = 0, piece = 0;
        bool more = walk.next(a), fresh = true;           // `fresh`: the next scores are a stretch's first
        int start = walk.t;
        uint32_t firsts = 0;                               // bit per score buffer: whether its tile's value product starts an output
        uint32_t idle = 0;
        long long since = 0;
        while (more || done < g) {
            // what is there: the groups of tile `g` (bits 0 to 4), the weights of tile `done` (5), the stretch's queries (6)
            uint64_t* look = lane < kGroups ? &bar.full[g & 1][lane] : (lane == 5 ? &bar.p_full : &bar.q_full);
            const int phase = lane < kGroups ? g >> 1 : (lane == 5 ? done : piece);
            const uint32_t there = __ballot_sync(0xffffffffu, mbar_test_wait(look, phase & 1));
            bool moved = false;
            if (done < g && (there >> 5 & 1) != 0) {
                fence_after();
                const uint32_t adds = (firsts >> (done & 1) & 1) ^ 1;
                if ((done & 1) == 0) values(std::integral_constant<int, 0>{}, adds);
                else values(std::integral_constant<int, 1>{}, adds);
                commit(&bar.o_done, leader);
                ++done;
                moved = true;
            }
            if (more && g <= done + 1 && (!fresh || group_of > 0 || (there >> 6 & 1) != 0) && (there >> group_of & 1) != 0) {
                fence_after();
                if ((g & 1) == 0) scores(std::integral_constant<int, 0>{}, there, group_of);
                else scores(std::integral_constant<int, 1>{}, there, group_of);
                if (group_of == kGroups) {
                    commit(&bar.s_full[g & 1], leader);
                    commit(&bar.empty[g & 1][kGroups - 1], leader);
                    firsts = (firsts & ~(1u << (g & 1))) | (uint32_t)fresh << (g & 1);
                    group_of = 0;
                    fresh = false;
                    ++g;
                    if (++walk.t == walk.until) {
                        commit(&bar.q_empty, leader);
                        walk.left -= walk.until - start;
                        more = walk.next(a);
                        start = walk.t;
                        fresh = true;
                        ++piece;
                    }
                }
                moved = true;
            }
            if (moved) {
                idle = 0;
            } else if ((++idle & 255u) == 0) {
                const long long now = clock64();
                if (idle == 256u) since = now;
                bool ok = *reinterpret_cast<volatile int*>(&bar.abort) == 0;
                if (now - since > kWaitCycles) ok = give_up(&bar.abort);
                if (!__all_sync(0xffffffffu, ok)) break;
            }
        }
        commit(&bar.drained, leader);
        drain(&bar.drained, 0);
        __syncwarp();
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
                float m[2], most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 32; i += 2) most[(i >> 1) & 3] = fmaxf(fmaxf(f(s[i]), f(s[i + 1])), most[(i >> 1) & 3]);
                m[0] = fmaxf(most[0], most[2]);
                m[1] = fmaxf(most[1], most[3]);
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
            if (whole) {
                // 16 dimensions x 32 rows at a time as fragments, stored transposed: a row's 32 dimensions of the warp leave as 64 bytes
                uint8_t* stage = p_smem + warp * 2048;   // [32 rows][64 bytes], the weights' place
                const int token = (lane & 7) + ((lane >> 4) << 3);
                __nv_bfloat16* dst = a.out + (int64_t)walk.b * a.out_batch + (int64_t)(rt * kRows) * a.out_row + warp * 32;
#pragma unroll 1
                for (int k = 0; k < 8; ++k) {
                    const int r0 = (k & 1) * 32;
#pragma unroll
                    for (int up = 0; up < 2; ++up) {
                        uint32_t o[16];
                        ld_frag32(tmem + kO + k * 32 + lanes + ((uint32_t)(up * 16) << 16), o);
                        wait_ld();
#pragma unroll
                        for (int i = 0; i < 2; ++i) {   // 16 rows
                            uint32_t y[4];
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const float2 e = *reinterpret_cast<const float2*>(&bar.factor[r0 + i * 16 + j * 8 + 2 * tc]);
                                const uint32_t* x = o + 8 * i + 4 * j;
                                y[2 * j] = pack_bf2(f(x[0]) * e.x, f(x[1]) * e.y);
                                y[2 * j + 1] = pack_bf2(f(x[2]) * e.x, f(x[3]) * e.y);
                            }
                            const int to = i * 16 + token, unit = up * 2 + ((lane >> 3) & 1);
                            asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(smem_u32(stage + to * 64 + ((unit ^ ((to >> 1) & 3)) << 4))), "r"(y[0]),
                                         "r"(y[1]), "r"(y[2]), "r"(y[3]) : "memory");
                        }
                    }
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int row_of = i * 8 + (lane >> 2), unit = lane & 3;
                        const uint4 x = *reinterpret_cast<const uint4*>(stage + row_of * 64 + ((unit ^ ((row_of >> 1) & 3)) << 4));
                        if (rt * kRows + r0 + row_of < a.R) *reinterpret_cast<uint4*>(dst + (int64_t)(r0 + row_of) * a.out_row + (k >> 1) * 128 + unit * 8) = x;
                    }
                    __syncwarp();
                }
            } else {
                const int rows = min(kRows, a.R - rt * kRows);
#pragma unroll 1
                for (int k = 0; k < 8; ++k) {
                    const int r0 = (k & 1) * 32;
                    if (r0 >= rows) continue;
                    uint32_t o[32];
                    ld32(tmem + kO + k * 32 + lanes, o);
                    wait_ld();
                    float* to = part + r0 * kValue + (k >> 1) * 128 + warp * 32 + lane;
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (r0 + j < rows) to[j * kValue] = f(o[j]) * bar.factor[r0 + j];
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

// Joins the parts of the sequences that a cut runs through: sum of w_p O_p over the parts, w_p = exp(lse_p - lse).  A CTA has some rows of a
// sequence, a lane 16 dimensions: as many warps share a row, taking its parts in turn, as there are parts.  One row and 16 warps, so that many
// parts of few rows are joined soon, or four rows and eight warps, four CTAs per SM, where there are more rows than that.
template <int kRowsEach, int kJoinWarps>
__global__ void __launch_bounds__(32 * kJoinWarps, kRowsEach == 1 ? 1 : 4) latent_join_kernel(const __grid_constant__ DecodeArgs a, int ctas, int per) {
    __shared__ float4 sums[kJoinWarps][kValue / 4];
    grid_dep_launch();
    grid_dep_wait();
    const int b = (int)blockIdx.x / per, r0 = ((int)blockIdx.x - b * per) * kRowsEach, end = min(a.R, r0 + kRowsEach);
    const int4 span = a.spans[b];
    const int first = span.x, parts = span.y - span.x + 1;
    if (parts == 1) return;   // (written by the one CTA that had it, or empty)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int sharing = kRowsEach == 1 || parts > 4 ? kJoinWarps : (parts > 2 ? 4 : 2), mine = warp % sharing;
    const float* lses = a.parts + (int64_t)ctas * 2 * kRows * kValue;
    for (int base = r0; base < end; base += kJoinWarps / sharing) {   // (all threads come as often to the barriers)
        const int r = base + warp / sharing, rt = r / kRows;
        // a CTA's first stretch is its slot 0
        auto slot = [&](int p) { return ((int64_t)((first + p) * a.row_tiles + rt) * 2 + (p > 0 || span.z != 0 ? 0 : 1)) * kRows + r % kRows; };
        float ref = -INFINITY, sum = 0.0f;
        float4 acc[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (r < end) {
            float4 next[4];   // (on their way while the weights are being made)
            if (mine < parts) {
#pragma unroll
                for (int k = 0; k < 4; ++k) next[k] = *reinterpret_cast<const float4*>(a.parts + slot(mine) * kValue + k * 128 + lane * 4);
            }
            const float first_lse = lane < parts ? lses[slot(lane)] : -INFINITY;
            ref = first_lse;
            for (int p = lane + 32; p < parts; p += 32) ref = fmaxf(ref, lses[slot(p)]);
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1) ref = fmaxf(ref, __shfl_xor_sync(0xffffffffu, ref, off));
            if (ref == -INFINITY) ref = 0.0f;
            const float first_weight = expf(first_lse - ref);   // (0 where there is no such part)
            sum = first_weight;
            for (int p = lane + 32; p < parts; p += 32) sum += expf(lses[slot(p)] - ref);
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
            for (int p = mine; p < parts; p += sharing) {
                float4 v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = next[k];
                if (p + sharing < parts) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) next[k] = *reinterpret_cast<const float4*>(a.parts + slot(p + sharing) * kValue + k * 128 + lane * 4);
                }
                const float w = p < 32 ? __shfl_sync(0xffffffffu, first_weight, p) : expf(lses[slot(p)] - ref);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    acc[k].x += w * v[k].x;
                    acc[k].y += w * v[k].y;
                    acc[k].z += w * v[k].z;
                    acc[k].w += w * v[k].w;
                }
            }
        }
        if (mine != 0) {
#pragma unroll
            for (int k = 0; k < 4; ++k) sums[warp][k * 32 + lane] = acc[k];
        }
        __syncthreads();
        if (mine == 0 && r < end) {
            const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                for (int x = 1; x < sharing; ++x) {
                    const float4 v = sums[warp + x][k * 32 + lane];
                    acc[k].x += v.x;
                    acc[k].y += v.y;
                    acc[k].z += v.z;
                    acc[k].w += v.w;
                }
                *reinterpret_cast<uint2*>(a.out + (int64_t)b * a.out_batch + (int64_t)r * a.out_row + k * 128 + lane * 4) =
                    make_uint2(pack_bf2(acc[k].x * inv, acc[k].y * inv), pack_bf2(acc[k].z * inv, acc[k].w * inv));
            }
            if (lane == 0 && a.lse != nullptr) a.lse[(int64_t)b * a.R + r] = sum == 0.0f ? -INFINITY : ref + logf(sum);
        }
        __syncthreads();
    }
}

int groups_for(int64_t row_tiles) {
    const int sms = device_sm_count();
    return row_tiles >= sms ? 1 : (int)(sms / row_tiles);
}

}  // namespace

size_t latent_decode_workspace(const fkda_latent_decode_params& p) {
    const int64_t row_tiles = (p.Tq * p.H + kRows - 1) / kRows;
    return (size_t)(row_tiles * groups_for(row_tiles)) * 2 * kRows * (kValue + 1) * sizeof(float) + (size_t)p.B * sizeof(int4);
}

int launch_latent_decode(const fkda_latent_decode_params& p, cudaStream_t stream, int* n_launches) {
    if (p.B > kMaxSeqs) return FKDA_ERR_BAD_SHAPE;
    DecodeArgs a;
    a.out = static_cast<__nv_bfloat16*>(p.out);
    a.lse = p.lse;
    a.table = p.block_table;
    a.cache = static_cast<const __nv_bfloat16*>(p.cache);
    a.page_stride = p.cache_stride[1] == kWidth ? p.cache_stride[0] : 0;
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
    a.starve_ms = starve_next();
    a.spans = reinterpret_cast<int4*>(a.parts + (int64_t)a.row_tiles * a.groups * 2 * kRows * (kValue + 1));
    DecodeMaps maps;
    const cuuint64_t qdims[3] = {(cuuint64_t)kWidth, (cuuint64_t)a.R, (cuuint64_t)p.B};
    const cuuint64_t qstrides[2] = {(cuuint64_t)p.q_stride[1] * 2, (cuuint64_t)p.q_stride[0] * 2};
    const cuuint32_t qbox[3] = {64u, (cuuint32_t)kRows, 1u};
    const cuuint64_t cdims[3] = {(cuuint64_t)kWidth, (cuuint64_t)p.page_size, (cuuint64_t)p.pages};
    const cuuint64_t cstrides[2] = {(cuuint64_t)p.cache_stride[1] * 2, (cuuint64_t)p.cache_stride[0] * 2};
    const cuuint32_t cbox[3] = {64u, (cuuint32_t)a.box, 1u};
    if (!encode_bf16_map(&maps.q, 3, p.q, qdims, qstrides, qbox)) return FKDA_ERR_LAUNCH;
    maps.cache = maps.q;   // (where there is no page, nothing is read)
    if (p.pages > 0 && p.max_pages > 0 && !encode_bf16_map(&maps.cache, 3, p.cache, cdims, cstrides, cbox)) return FKDA_ERR_LAUNCH;
    const int ctas = a.row_tiles * a.groups;
    // Both shapes, one row a CTA against four: 16 sequences of 32 heads (512 rows) up to 3 000 tokens 26.2 us against 35.1, one of 64
    // heads up to 20 000 19.8 against 71.5; 64 of 16 heads (1 024 rows) 58.8 against 53.4, 16 of 64 heads (1 024) 34.9 against 37.9; 32 of
    // 64 heads (2 048) 58.4 against 47.6, 64 of 128 heads (8 192) 169 against 90.
    const int rows_each = p.B * a.R > 4 * device_sm_count() ? 4 : 1, per = (a.R + rows_each - 1) / rows_each;
    const int64_t joins = p.B * per;
    if (joins > 0x7fffffff) return FKDA_ERR_BAD_SHAPE;
    if (!allow_smem<latent_decode_kernel>(kSmem)) return FKDA_ERR_LAUNCH;
    if (!launch_dependent(latent_decode_kernel, ctas, kThreads, kSmem, stream, a, maps)) return FKDA_ERR_LAUNCH;
    if (!(rows_each == 1 ? launch_dependent(latent_join_kernel<1, 16>, joins, 512, 0, stream, a, ctas, per)
                         : launch_dependent(latent_join_kernel<4, 8>, joins, 256, 0, stream, a, ctas, per)))
        return FKDA_ERR_LAUNCH;
    *n_launches = 2;
    return FKDA_OK;
}

int decode_gave_up(cudaStream_t stream, uint32_t* times) { return read_gave_up(stream, times); }

}  // namespace fkda
