// Inline-PTX wrappers for tensor memory and tcgen05.mma, and the waits of the kernels that use them (linear and latent
// attention).
#pragma once

#include "fkda_common.cuh"
#include "fkda_internal.h"
#include "fkda_sm100.cuh"

namespace fkda {
namespace tc5 {

using namespace sm100;

// ------------------------------------------------------------------ waits ----
// Every wait of these kernels is bounded.  One that gives up raises the CTA's abort flag, at which the other waits of the CTA return
// soon: no more copies are issued, the other roles run to their ends on whatever is in shared memory (all accesses in bounds), what is
// in flight is waited for, tensor memory is freed, and the count below tells the host (fkda_operator_status).
static __device__ uint32_t g_gave_up = 0;
// The limit is counted in SM cycles (two seconds at 2 GHz): the global timer is far away, and reading it in the waits of a dozen
// warps made all of them slower.
constexpr long long kWaitCycles = 4000000000ll;

// Not inlined: thirty copies of it leave the roles' loops less room in the instruction cache.  (Except where a role takes nearly all
// registers that a thread can have: a call has its own there.)
#ifdef FKDA_WAITS_INLINE
#define FKDA_WAIT_INLINE __forceinline__
#else
#define FKDA_WAIT_INLINE __noinline__
#endif
static __device__ FKDA_WAIT_INLINE bool wait_on(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
    long long start = 0;
    for (uint32_t spins = 0; !mbar_try_wait(bar, parity); ++spins) {
        if ((spins & 31u) != 31u) continue;
        if (abort_flag != nullptr && *abort_flag != 0) return false;
        const long long now = clock64();
        if (start == 0) start = now;
        if (now - start > kWaitCycles) return false;
    }
    return true;
}
__device__ __forceinline__ bool wait_until(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
    return mbar_try_wait(bar, parity) || wait_on(bar, parity, abort_flag);
}

// How often this translation unit's kernels have given up on the current device, once the stream has come this far.  Only ever counted
// up: several threads may ask, and kernels on other streams may give up meanwhile.
static int read_gave_up(cudaStream_t stream, uint32_t* times) {
    const bool read = cudaMemcpyFromSymbolAsync(times, g_gave_up, sizeof(*times), 0, cudaMemcpyDeviceToHost, stream) == cudaSuccess;
    return read && cudaStreamSynchronize(stream) == cudaSuccess ? FKDA_OK : FKDA_ERR_LAUNCH;
}

static __device__ FKDA_WAIT_INLINE bool give_up(int* abort_flag) {
    *reinterpret_cast<volatile int*>(abort_flag) = 1;
    atomicAdd(&g_gave_up, 1u);
    return false;
}
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, int* abort_flag) {
    return wait_until(bar, parity, abort_flag) || give_up(abort_flag);
}
// For a stage that the next copies go to.  A role that has given up runs on and frees stages whose last copies may still be on their way;
// their barrier must not be armed a second time in one phase, so no more copies are issued then.
__device__ __forceinline__ bool wait_free(uint64_t* bar, uint32_t parity, int* abort_flag) {
    return wait(bar, parity, abort_flag) && *reinterpret_cast<volatile int*>(abort_flag) == 0;
}
// TEST ONLY: what a loading warp does in a call that is to starve: nothing is loaded, its own wait for the first tile runs out after so many
// milliseconds (at some 2 cycles per ns), and the other roles' waits end by the flag.
static __device__ __noinline__ void starve(uint64_t* bar, int ms, int* abort_flag) {
    const long long start = clock64();
    while (!mbar_try_wait(bar, 0) && clock64() - start < ms * 2000000ll) {}
    give_up(abort_flag);
    __syncwarp();
}
// The same for a whole warp, whose lanes leave it together: what follows may be an access to tensor memory or another instruction that
// a warp executes as one.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, int* abort_flag) {
    const bool ok = wait(bar, parity, abort_flag);
    __syncwarp();
    return ok;
}
// For what is in flight when a role ends: not cut short by the abort flag.
__device__ __forceinline__ void drain(uint64_t* bar, uint32_t parity) { wait_until(bar, parity, nullptr); }

__device__ __forceinline__ void arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void named_sync(int id, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
// Barrier among `threads` threads that tells all of them whether any had `x` true.
__device__ __forceinline__ bool named_any(int id, int threads, bool x) {
    uint32_t any;
    asm volatile(
        "{\n.reg .pred p, q;\nsetp.ne.u32 p, %3, 0;\nbarrier.cta.red.or.pred q, %1, %2, p;\nselp.u32 %0, 1, 0, q;\n}\n"
        : "=r"(any)
        : "r"(id), "r"(threads), "r"((uint32_t)x)
        : "memory");
    return any != 0;
}

// Copies are issued by the lane with `leader` = 1 of a warp that runs the code around them as a whole, as products are (below).
__device__ __forceinline__ void expect(uint64_t* bar, uint32_t bytes, uint32_t leader) {
    asm volatile("{\n.reg .pred q;\nsetp.ne.b32 q, %2, 0;\n@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n}\n" ::"r"(smem_u32(bar)), "r"(bytes), "r"(leader) : "memory");
}
__device__ __forceinline__ void load_4d(uint32_t dst, const void* tmap, int c0, int c1, int c2, int c3, uint64_t* bar, uint32_t leader) {
    asm volatile(
        "{\n.reg .pred q;\nsetp.ne.b32 q, %7, 0;\n"
        "@q cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];\n}\n" ::"r"(dst), "l"(tmap),
        "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar)), "r"(leader)
        : "memory");
}
__device__ __forceinline__ void load_3d(uint32_t dst, const void* tmap, int c0, int c1, int c2, uint64_t* bar, uint32_t leader) {
    asm volatile(
        "{\n.reg .pred q;\nsetp.ne.b32 q, %6, 0;\n"
        "@q cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n}\n" ::"r"(dst), "l"(tmap),
        "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar)), "r"(leader)
        : "memory");
}
__device__ __forceinline__ void tma_store_4d(const void* tmap, int c0, int c1, int c2, int c3, const void* smem_src) {
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(tmap), "r"(c0), "r"(c1), "r"(c2),
                 "r"(c3), "r"(smem_u32(smem_src))
                 : "memory");
}

// ---------------------------------------------------------- tensor memory ----
// One full warp allocates `n_cols` (power of two, 32..512) columns; the base address is written to shared memory.  The same
// warp frees them before the CTA exits.
__device__ __forceinline__ void tmem_alloc(uint32_t* smem_result, uint32_t n_cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(smem_result)), "r"(n_cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t n_cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(n_cols) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Each thread reads or writes its own lane (lane field of taddr = 32 * (warp % 4)), 32 consecutive 32-bit columns.
__device__ __forceinline__ void ld32(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void st32(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void st16(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
                 "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
// Fragment-shaped accesses of 16 lanes, for accumulators of 64 rows (rows 16 w .. 16 w + 15 live in lanes 32 w .. 32 w + 15) and for
// operands that arrive in fragments.  Thread 4 g + t of the warp:
//   load of 8 n columns:  r[4 i], r[4 i + 1] = (lane g, columns 8 i + 2 t, + 1), r[4 i + 2], r[4 i + 3] = (lane g + 8, the same)
//   store of 8 columns:   r[0], r[1] -> (lanes g and g + 8, column t), r[2], r[3] -> (lanes g and g + 8, column 4 + t)
// The store's registers are those of an mma.sync A fragment, or of transposed 8 x 8 blocks as ldmatrix loads them: pairs of bf16
// along K, as an A operand in tensor memory has them.
__device__ __forceinline__ void ld_frag16(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void ld_frag32(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void ld_frag64(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void st_frag8(uint32_t taddr, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
    asm volatile("tcgen05.st.sync.aligned.16x128b.x2.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr), "r"(r0), "r"(r1), "r"(r2), "r"(r3) : "memory");
}

// The kernels count on dynamic shared memory that starts at a multiple of 1024 bytes, as it is declared, and on tensor memory that starts
// at 0 where a CTA has all of it: then addresses and descriptors are constants.  (Never seen otherwise; checked all the same.)
__device__ __forceinline__ bool as_assumed(const void* smem, uint32_t tmem) {
    if ((smem_u32(smem) & 1023u) == 0 && tmem == 0) return true;
    atomicAdd(&g_gave_up, 1u);
    return false;
}

// A warpgroup's registers per thread from here on: `inc` waits until others have given up as many (the shares of all warpgroups of a
// block may not add up to more than it was launched with).
template <int N>
__device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// Pairs of fp32 in one instruction.
__device__ __forceinline__ void fma2(uint32_t& x, uint32_t& y, float b, float c) {   // x b + c, y b + c
    asm("{\n.reg .b64 a, b, c;\nmov.b64 a, {%0,%1};\nmov.b64 b, {%2,%2};\nmov.b64 c, {%3,%3};\nfma.rn.ftz.f32x2 a, a, b, c;\nmov.b64 {%0,%1}, a;\n}\n"
        : "+r"(x), "+r"(y)
        : "f"(b), "f"(c));
}
__device__ __forceinline__ void add2(float& x, float& y, uint32_t bx, uint32_t by) {
    asm("{\n.reg .b64 a, b;\nmov.b64 a, {%0,%1};\nmov.b64 b, {%2,%3};\nadd.rn.ftz.f32x2 a, a, b;\nmov.b64 {%0,%1}, a;\n}\n" : "+f"(x), "+f"(y) : "r"(bx), "r"(by));
}
__device__ __forceinline__ void mul2(uint32_t& x, uint32_t& y, float bx, float by) {
    asm("{\n.reg .b64 a, b;\nmov.b64 a, {%0,%1};\nmov.b64 b, {%2,%3};\nmul.rn.ftz.f32x2 a, a, b;\nmov.b64 {%0,%1}, a;\n}\n" : "+r"(x), "+r"(y) : "f"(bx), "f"(by));
}
__device__ __forceinline__ void sub2(uint32_t& x, uint32_t& y, uint32_t bx, uint32_t by) {   // x - b: the signs of b flipped by a product with -1
    asm("{\n.reg .b64 a, b, m;\nmov.b64 a, {%0,%1};\nmov.b64 b, {%2,%3};\nmov.b64 m, {%4,%4};\nfma.rn.ftz.f32x2 a, b, m, a;\nmov.b64 {%0,%1}, a;\n}\n"
        : "+r"(x), "+r"(y)
        : "r"(bx), "r"(by), "f"(-1.0f));
}

// ------------------------------------------------------------ tcgen05.mma ----
// Shared-memory operands are tiles of 128-byte rows (64 bf16), written by tiled copies with the 128-byte swizzle (the 16-byte
// pieces of row r are permuted by r % 8); tiles start at multiples of 1024 bytes.
//   K-major operand: a tile row is a row of the operand, the tile's columns are 64 steps of K; 16 steps are 32 bytes of the start
//     address; groups of 8 rows are 1024 bytes apart.
//   MN-major operand: a tile row is one step of K, the tile's columns are 64 rows (M or N) of the operand; 16 steps are 2048 bytes
//     of the start address; `block` is the distance to the tile of the next 64 rows.
// Fields: start address [0,14), leading distance [16,30), stride of 8-row groups [32,46) (all >> 4), version 1 at bit 46,
// swizzle mode 2 (128 bytes) at [61,64).  The upper word is the same for all; this is the lower one.
constexpr uint32_t kDescUpper = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc(uint32_t smem_addr, uint32_t block = 16) { return ((smem_addr >> 4) & 0x3fffu) | ((block >> 4) << 16); }
// Instruction descriptor for bf16 operands and fp32 accumulation: D format [4,6) = 1, A and B formats [7,10), [10,13) = 1, MN-major
// flags of A and B at bits 15 and 16, N >> 3 at [17,23), M >> 4 at [24,29).
__host__ __device__ constexpr uint32_t idesc(int M, int N, bool a_mn, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) |
           ((uint32_t)(M >> 4) << 24);
}
// Products are issued by ONE thread, but a whole warp runs the code around them, with the same values in all lanes: measured so, an
// instruction goes out every 32 to 64 cycles (what its operands take) instead of every 75 (A in tensor memory) or 116, probably because
// descriptors then need not be moved for each.  `leader` is 1 in the lane that issues.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }
// D[tmem] (+)= A[smem] B[smem], K = 16; accumulate = 0 overwrites D.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t accumulate, uint32_t leader) {
    asm volatile(
        "{\n.reg .pred p, q;\n.reg .b64 da, db;\nmov.b64 da, {%1, %5};\nmov.b64 db, {%2, %5};\nsetp.ne.b32 p, %4, 0;\nsetp.ne.b32 q, %6, 0;\n"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}\n" ::"r"(d), "r"(a), "r"(b), "r"(id), "r"(accumulate), "r"(kDescUpper), "r"(leader)
        : "memory");
}
// D[tmem] (+)= A[tmem] B[smem]: A sits in tensor memory, two bf16 per 32-bit column (8 columns per instruction).
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t accumulate, uint32_t leader) {
    asm volatile(
        "{\n.reg .pred p, q;\n.reg .b64 db;\nmov.b64 db, {%2, %5};\nsetp.ne.b32 p, %4, 0;\nsetp.ne.b32 q, %6, 0;\n"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}\n" ::"r"(d), "r"(a), "r"(b), "r"(id), "r"(accumulate), "r"(kDescUpper), "r"(leader)
        : "memory");
}
// The mbarrier completes when all tcgen05.mma issued so far by the leader have.
__device__ __forceinline__ void commit(uint64_t* bar, uint32_t leader) {
    asm volatile("{\n.reg .pred q;\nsetp.ne.b32 q, %1, 0;\n@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar)),
                 "r"(leader)
                 : "memory");
}

__device__ __forceinline__ float f(uint32_t x) { return __uint_as_float(x); }
__device__ __forceinline__ uint32_t u(float x) { return __float_as_uint(x); }

}  // namespace tc5
}  // namespace fkda
