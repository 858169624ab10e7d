/*
 * Block-scaled fp8 product on Blackwell tensor cores (sm_100a):
 *   D[m][n] = C[m][n] + sum over blocks kb of 128 k of  sA[m][kb] sB[n][kb] sum_{k in kb} A[m][k] B[n][k].
 *
 * Shape of the kernel
 *  - A k-block is 128 codes = 128 bytes: one row of the copy engine's 128-byte swizzle and one block of the scales, so
 *    a stage of the shared-memory ring, an accumulation of the tensor core and a pair of scales are the same step.
 *  - tcgen05.mma kind::f8f6f4 sums the 128 products of a k-block in tensor memory (fp32); the epilogue warps fetch the
 *    finished block, multiply it by both scales and add it to a running sum in registers with IEEE fp32 arithmetic,
 *    while the tensor core works on the next block in the other of two buffers.  So scales may be any fp32 numbers,
 *    and the tensor core's own accumulator (which rounds toward zero) never sums more than 128 values.
 *  - Warp-specialised, persistent: warp 0 = TMA producer, warp 1 = MMA issuer and tensor-memory owner, warp 2 = scale
 *    loader (cp.async into a ring of its own, eight k-blocks ahead), warps 4..11 = epilogue (four lane quarters x two
 *    column halves).  Roles are whole warps whose control flow the compiler can see to be uniform (the warp's number
 *    comes from a shuffle, waits end in a vote, one elected lane issues): with a single thread's flow instead, every
 *    operand of an MMA is moved to a uniform register first and a k-block costs about 500 clocks to issue, 264 so.
 *  - The commit of a k-block's MMAs says two things at once, that its stage may be refilled and that its sum is
 *    ready: producer and epilogue wait on the same barrier.
 *  - Every wait on an mbarrier is bounded; on expiry the waiter records where it gave up in the context's status word,
 *    all roles drain and the kernel returns.
 */
#include "fp8.cuh"
#include "tc_ptx.cuh"

#include <cudaTypedefs.h>

#include <mutex>

namespace {

using namespace tcptx;
using namespace fp8;

constexpr int BM_CTA = 128;        /* rows of A (and accumulator lanes) per CTA      */
constexpr int BK = 128;            /* codes per k-block                               */
constexpr int THREADS = 384;
constexpr int EPI_WARPS = 8;
constexpr int SLOTS = 8;           /* k-blocks in the scale ring                       */
constexpr int SMEM_LIMIT = 232448;

struct ScaleView {                 /* scale of row r, k-block kb: p[(r >> shift) * rs + kb * ks]  */
    const float* p;
    int64_t rs, ks;
    int shift;
};

struct Params {
    int64_t M, N;
    int tiles_m, tiles_n, num_kb, tile_group;
    uint32_t idesc;
    ScaleView sa, sb;
    const void* C; int64_t ldc;
    void* D; int64_t ldd;
    int d_type;
    bool tma_store;                /* D leaves, and C comes, through the copy engine   */
    bool d_vec;                    /* four results of a row may leave in one store      */
    Waits waits;                   /* (of the tile that is `lost` the last k-block is never brought) */
};

/* True in one lane of a converged warp, always the same one. */
__device__ __forceinline__ bool elect_one()
{
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

/* Bounded wait of a whole warp; false, for all its lanes, when it gave up or another role already had.  The timer, whose
 * read costs more than a k-block's arithmetic, is looked at only once a wait has lasted a thousand tries. */
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, const Params& p, int where, int detail)
{
    unsigned long long t0 = 0;
    for (uint32_t spins = 1; !__all_sync(0xffffffffu, mbar_try_wait(bar, parity)); ++spins) {
        if ((spins & 1023u) == 0) {
            bool over = false;
            if (elect_one()) {
                const unsigned long long t = globaltimer_ns();
                if (t0 == 0) t0 = t;
                over = gave_up(p.waits);
                if (!over && (long long)(t - t0) > p.waits.limit_ns) {
                    over = true;
                    give_up(p.waits, where, detail);
                }
            }
            if (__any_sync(0xffffffffu, over)) return false;
        }
    }
    return true;
}

/* When the issuer leaves early: waits (with a limit) for the commit of its last k-block, whose matrix instructions may still be at work
 * on tensor memory that is about to be given back. */
__device__ __forceinline__ void drain_mma(uint32_t bar, uint32_t parity)
{
    for (int tries = 0; tries < 2048 && !mbar_try_wait(bar, parity); ++tries) __nanosleep(64);
}

/* A k-block: four steps of 32 codes (two units of 16 bytes in a descriptor), the first overwriting the accumulator, and the commit, by
 * one elected lane of a converged warp.  In one piece under one predicate: 1 x 4096 x 4096 5.94 us with a branch around the steps, 5.64
 * so; in the pairs' kernel no difference. */
template <int CTAS>
__device__ __forceinline__ void umma_block(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t bar)
{
#define STEP(P, A, B, G) "@e tcgen05.mma.cta_group::" G ".kind::f8f6f4 [%0], " A ", " B ", %3, " P ";\n\t"
    if (CTAS == 1)
        asm volatile("{\n\t.reg .pred e, f, t;\n\tsetp.ne.b32 f, 0, 0;\n\tsetp.eq.b32 t, 0, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
                     STEP("f", "%1", "%2", "1") STEP("t", "%5", "%6", "1") STEP("t", "%7", "%8", "1") STEP("t", "%9", "%10", "1")
                     "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%4];\n\t}"
                     :: "r"(tmem_d), "l"(a), "l"(b), "r"(idesc), "r"(bar), "l"(a + 2), "l"(b + 2), "l"(a + 4), "l"(b + 4), "l"(a + 6), "l"(b + 6) : "memory");
    else
        asm volatile("{\n\t.reg .pred e, f, t;\n\tsetp.ne.b32 f, 0, 0;\n\tsetp.eq.b32 t, 0, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
                     STEP("f", "%1", "%2", "2") STEP("t", "%5", "%6", "2") STEP("t", "%7", "%8", "2") STEP("t", "%9", "%10", "2")
                     "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%4], %11;\n\t}"
                     :: "r"(tmem_d), "l"(a), "l"(b), "r"(idesc), "r"(bar), "l"(a + 2), "l"(b + 2), "l"(a + 4), "l"(b + 4), "l"(a + 6), "l"(b + 6),
                        "h"((uint16_t)3) : "memory");
#undef STEP
}

/* fp32 accumulator; operand formats e4m3 = 0, e5m2 = 1 at bits 7-9 and 10-12; both K-major. */
uint32_t make_idesc_fp8(int umma_m, int umma_n, int a_type, int b_type)
{
    return (1u << 4) | ((uint32_t)a_type << 7) | ((uint32_t)b_type << 10) | ((uint32_t)(umma_n >> 3) << 17) | ((uint32_t)(umma_m >> 4) << 24);
}

/* Asynchronous copy of one scale; `ok` false writes zero.  The mbarrier arrival follows this thread's copies. */
__device__ __forceinline__ void cp_async4(uint32_t dst, const float* src, bool ok)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" :: "r"(dst), "l"(src), "r"(ok ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint32_t bar)
{
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" :: "r"(bar) : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint32_t bar)
{
    asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" :: "r"(bar) : "memory");
}
/* One elected lane of a converged warp arrives on a barrier of the cluster and on one of its own CTA.  What the first releases are
 * reads of tensor memory, which tcgen05.wait::ld and the tcgen05 fence before it have ordered; a release at cluster scope would add
 * a memory fence of about a thousand clocks, twice a k-block's arithmetic.  Both CTAs of a pair address the leader's barrier the same
 * way and the lane is chosen by a predicate: with branches for either the warp's next wait began later, and 4096 x 4096 x 8192
 * took 184 us (a factor per row) and 129 (one per block), so 164 and 122. */
__device__ __forceinline__ void mbar_arrive_both(uint32_t bar_cluster, uint32_t bar)
{
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\t"
                 "@p mbarrier.arrive.shared::cluster.b64 _, [%0];\n\t"
                 "@p mbarrier.arrive.release.cta.shared::cta.b64 _, [%1];\n\t}" :: "r"(bar_cluster), "r"(bar) : "memory");
}

__device__ __forceinline__ void sts_u32(uint32_t at, uint32_t v) { asm volatile("st.shared.u32 [%0], %1;" :: "r"(at), "r"(v) : "memory"); }
/* From the shared memory of a CTA of the cluster (this one's included). */
__device__ __forceinline__ uint32_t lds_cluster_u32(uint32_t at)
{
    uint32_t v; asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory"); return v;
}
__device__ __forceinline__ float lds_f32(uint32_t at)
{
    float v; asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory"); return v;
}

__device__ __forceinline__ float2 lds_f32x2(uint32_t at)
{
    float2 v; asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory"); return v;
}
/* From the shared memory of a CTA of the cluster. */
__device__ __forceinline__ float4 lds_cluster_f32x4(uint32_t at)
{
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}

__device__ __forceinline__ float4 lds_f32x4(uint32_t at)
{
    float4 v; asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory"); return v;
}

/* 16 lanes x 8 G columns: register 4 g + k is column 8 g + 2 (lane % 4) + (k & 1) of lane lane / 4 + 8 (k >> 1). */
template <int G>
__device__ __forceinline__ void tmem_ld_16x256(uint32_t taddr, float* v)
{
    if constexpr (G == 1)
        asm volatile("tcgen05.ld.sync.aligned.16x256b.x1.b32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(taddr) : "memory");
    else if constexpr (G == 2)
        asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]) : "r"(taddr) : "memory");
    else
        asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                     : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
                       "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ uint64_t lds_b64(uint32_t at)
{
    uint64_t v; asm volatile("ld.shared.b64 %0, [%1];" : "=l"(v) : "r"(at) : "memory"); return v;
}
/* tcgen05.wait::ld with the loaded registers as operands: nothing that reads them can be moved ahead of it. */
template <int N>
__device__ __forceinline__ void tmem_ld_wait_n(float* v)
{
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]) :: "memory");
#pragma unroll
    for (int i = 4; i < N; ++i) asm volatile("" : "+f"(v[i]) :: "memory");
}

/* Tile order: groups of `group` tile-rows, column by column inside a group (operand panels shared in L2). */
__device__ __forceinline__ void tile_coords(int t, int tiles_m, int tiles_n, int group, int& tm, int& tn)
{
    const int per_group = group * tiles_n, g = t / per_group, first_m = g * group;
    const int gsz = min(tiles_m - first_m, group), r = t - g * per_group;
    tm = first_m + r % gsz;
    tn = r / gsz;
}

/* 32 columns of a warp's 32 rows leave through the warp's 4 KiB box in shared memory: thread r holds row r, so its own
 * stores would touch 32 rows an instruction (8000 clocks for a warp's 128 columns, a sixth of a K = 8192 tile).
 * 16-byte pieces are XOR-ed with the row, which is the copy engine's 128-byte swizzle and keeps the banks apart.
 *
 * Through the copy engine: 16-byte pieces of this row from `first` on (8 of them fill the box), then one store of the box.
 * ADD: the box holds the addend, brought there by the copy engine before. */
template <typename T, bool ADD>
__device__ __forceinline__ void box_pieces(uint32_t box, int lane, int first, const float* v)
{
    constexpr int E = 16 / sizeof(T);
#pragma unroll
    for (int j = 0; j < 32; j += E) {
        const uint32_t at = box + (uint32_t)lane * 128u + (uint32_t)(((first + j / E) ^ (lane & 7)) << 4);
        uint4 u;
        T* e = reinterpret_cast<T*>(&u);
        if (ADD) asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(at) : "memory");
#pragma unroll
        for (int k = 0; k < E; ++k) e[k] = from_f32<T>(ADD ? v[j + k] + to_f32(e[k]) : v[j + k]);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" :: "r"(at), "r"(u.x), "r"(u.y), "r"(u.z), "r"(u.w) : "memory");
    }
}

/* The same from registers in the 16x256b shape (two lane halves of four groups of eight columns). */
template <typename T, bool ADD>
__device__ __forceinline__ void box_fragments(uint32_t box, int lane, int first, const float* v)
{
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
        const int r = (i >> 4) * 16 + ((i >> 1) & 1) * 8 + (lane >> 2), g = (i >> 2) & 3;
        const uint32_t row = box + (uint32_t)r * 128u;
        if constexpr (sizeof(T) == 4) {
            const uint32_t at = row + (uint32_t)(((2 * g + ((lane & 3) >> 1)) ^ (r & 7)) << 4) + (uint32_t)(lane & 1) * 8u;
            float2 c = make_float2(0.0f, 0.0f);
            if (ADD) c = lds_f32x2(at);
            asm volatile("st.shared.v2.f32 [%0], {%1, %2};" :: "r"(at), "f"(v[i] + c.x), "f"(v[i + 1] + c.y) : "memory");
        } else {
            const uint32_t at = row + (uint32_t)(((first + g) ^ (r & 7)) << 4) + (uint32_t)(lane & 3) * 4u;
            uint32_t u = 0;
            if (ADD) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(u) : "r"(at) : "memory");
            T* e = reinterpret_cast<T*>(&u);
            e[0] = from_f32<T>(ADD ? v[i] + to_f32(e[0]) : v[i]);
            e[1] = from_f32<T>(ADD ? v[i + 1] + to_f32(e[1]) : v[i + 1]);
            asm volatile("st.shared.b32 [%0], %1;" :: "r"(at), "r"(u) : "memory");
        }
    }
}
template <bool FRAGMENTS, bool ADD>
__device__ __forceinline__ void box_write(int type, uint32_t box, int lane, int first, const float* v)
{
    if constexpr (FRAGMENTS) {
        if (type == DECXB_F32)      box_fragments<float, ADD>(box, lane, first, v);
        else if (type == DECXB_F16) box_fragments<__half, ADD>(box, lane, first, v);
        else                        box_fragments<__nv_bfloat16, ADD>(box, lane, first, v);
    } else {
        if (type == DECXB_F32)      box_pieces<float, ADD>(box, lane, first, v);
        else if (type == DECXB_F16) box_pieces<__half, ADD>(box, lane, first, v);
        else                        box_pieces<__nv_bfloat16, ADD>(box, lane, first, v);
    }
}

/* By the threads, row after row with one column a lane: any address and pitch, and the addend on the way. */
template <typename T>
__device__ __forceinline__ void box_rows(const Params& p, uint32_t box, int lane, int64_t row0, int64_t col)
{
    if (col >= p.N) return;
    const int rows = (int)min((int64_t)32, p.M - row0);
    T* d = static_cast<T*>(p.D) + row0 * p.ldd + col;
    const T* c = p.C ? static_cast<const T*>(p.C) + row0 * p.ldc + col : nullptr;
#pragma unroll 8
    for (int r = 0; r < rows; ++r) {
        float v = lds_f32(box + (uint32_t)r * 128u + (uint32_t)(((lane >> 2) ^ (r & 7)) << 4) + (uint32_t)(lane & 3) * 4u);
        if (c) v += to_f32(c[(int64_t)r * p.ldc]);
        d[(int64_t)r * p.ldd] = from_f32<T>(v);
    }
}

/* Up to four adjacent results: (+C), one rounding, one store where the rows allow it. */
template <typename T>
__device__ __forceinline__ void put4(const Params& p, int64_t row, int64_t col, int have, float4 v)
{
    T* d = static_cast<T*>(p.D) + row * p.ldd + col;
    float f[4] = {v.x, v.y, v.z, v.w};
    if (p.C) {
        const T* c = static_cast<const T*>(p.C) + row * p.ldc + col;
#pragma unroll
        for (int j = 0; j < 4; ++j) if (j < have) f[j] += to_f32(c[j]);
    }
    if (have == 4 && p.d_vec) {
        alignas(16) T o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = from_f32<T>(f[j]);
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(d) = *reinterpret_cast<const uint4*>(o);
        else                          *reinterpret_cast<uint2*>(d) = *reinterpret_cast<const uint2*>(o);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) if (j < have) d[j] = from_f32<T>(f[j]);
    }
}

/* --------------------------------------------------------------------------------------
 * Many result tiles: a pair of CTAs (cta_group::2) per tile of 256 x 256, each with 128 rows of A and 128 of B.
 * 16384 x 4096 x 8192 takes 440 to 520 us (2.1 to 2.5 PFLOP/s, the SM clock near 1.55 GHz under the power cap). A k-block costs some 890
 * clocks of an SM where the tensor core needs 512: feeding the tiles alone takes 231 us of that size, the MMAs alone
 * about 440, reading tensor memory and adding alone 393, and the last two overlap only in part, two accumulators being
 * all that tensor memory holds. With a factor per column two operations an element, and what the
 * same warps wait between k-blocks, bound it: 1.67 PFLOP/s.
 * COLVEC : B has a scale per row (block_rows 1): each column of the tile has its own factor.  Otherwise a
 *          128-row block of B has one scale, and the columns of one epilogue warp lie in one block.
 * ADDEND : C comes through the copy engine into the boxes that the results leave from, the first of a tile during its
 *          product (4096 x 4096 x 8192 with an fp32 addend: 218 us, with the threads' own loads 436).
 * ------------------------------------------------------------------------------------ */
template <bool COLVEC>
struct Cfg {
    static constexpr int CTAS = 2;
    static constexpr int BN = 128;                             /* rows of B per CTA */
    static constexpr int UMMA_M = BM_CTA * CTAS;
    static constexpr int UMMA_N = BN * CTAS;
    static constexpr int ACC = UMMA_N / 2;                     /* columns per epilogue warp */
    static constexpr int A_BYTES = BM_CTA * BK;
    static constexpr int B_BYTES = BN * BK;
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int KB_FLOATS = BM_CTA + (COLVEC ? UMMA_N : 32);
    static constexpr int SCALE_BYTES = SLOTS * KB_FLOATS * 4;
    static constexpr int BOXES = 2;                            /* result boxes of a warp, one filled while the other is read */
    static constexpr int BOX_BYTES = EPI_WARPS * BOXES * 4096;
    static constexpr int STAGES = (SMEM_LIMIT - 2048 - SCALE_BYTES - BOX_BYTES) / STAGE_BYTES;
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + BOX_BYTES + SCALE_BYTES + 1024 /* alignment slack */ + 512 /* barriers */;
    static constexpr int BUFS = 512 / UMMA_N;                  /* accumulators in tensor memory */
    static constexpr int TMEM_COLS = BUFS * UMMA_N;
    static_assert(SMEM_BYTES <= SMEM_LIMIT, "shared memory");
    /* the epilogue reads a stage's barrier by parity and lies at most BUFS k-blocks behind the issuer */
    static_assert(STAGES > BUFS, "a stage's barrier must not turn over twice unseen");
};

template <bool COLVEC, bool ADDEND>
__global__ void __launch_bounds__(THREADS, 1)
decxb_gemm_fp8_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                      const __grid_constant__ CUtensorMap map_d, const __grid_constant__ CUtensorMap map_c, const Params p)
{
    using C = Cfg<COLVEC>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;     /* the swizzle is a function of address bits 4-9 */
    const uint32_t boxes = smem_base + C::STAGES * C::STAGE_BYTES;
    const uint32_t ring = boxes + C::BOX_BYTES;
    const uint32_t bars = ring + C::SCALE_BYTES;
    auto full_bar   = [&](int s) { return bars + 8u * s; };
    auto done_bar   = [&](int s) { return bars + 8u * (C::STAGES + s); };      /* MMAs of the stage finished */
    auto tempty_bar = [&](int b) { return bars + 8u * (2 * C::STAGES + b); };
    auto sfull_bar  = [&](int s) { return bars + 8u * (2 * C::STAGES + C::BUFS + s); };
    auto sempty_bar = [&](int s) { return bars + 8u * (2 * C::STAGES + C::BUFS + SLOTS + s); };
    auto addend_bar = [&](int w) { return bars + 8u * (2 * C::STAGES + C::BUFS + 2 * SLOTS + w); };       /* one a box */
    const uint32_t tmem_slot = bars + 8u * (2 * C::STAGES + C::BUFS + 2 * SLOTS + 2 * EPI_WARPS);
    auto stage_a = [&](int s) { return smem_base + s * C::STAGE_BYTES; };
    auto stage_b = [&](int s) { return smem_base + s * C::STAGE_BYTES + C::A_BYTES; };

    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t cta_rank = cluster_ctarank();
    const bool is_leader = cta_rank == 0;
    const int cluster_id = (int)blockIdx.x / C::CTAS, num_clusters = (int)gridDim.x / C::CTAS;
    const int num_tiles = p.tiles_m * p.tiles_n;

    if (threadIdx.x == 0) {
        prefetch_tensormap(&map_a); prefetch_tensormap(&map_b);
        if (p.tma_store) prefetch_tensormap(&map_d);
        if (ADDEND) prefetch_tensormap(&map_c);
        for (int s = 0; s < C::STAGES; ++s) { mbar_init(full_bar(s), 1); mbar_init(done_bar(s), 1); }
        for (int b = 0; b < C::BUFS; ++b) mbar_init(tempty_bar(b), EPI_WARPS * C::CTAS);
        for (int s = 0; s < SLOTS; ++s) { mbar_init(sfull_bar(s), 32); mbar_init(sempty_bar(s), EPI_WARPS); }
        for (int w = 0; w < 2 * EPI_WARPS; ++w) mbar_init(addend_bar(w), 1);
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc<C::CTAS>(tmem_slot, C::TMEM_COLS);
        tmem_relinquish<C::CTAS>();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    uint32_t tmem_base;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot));
    /* the next kernel of the stream may take this one's place as its blocks leave; this one starts on the memory of
     * the kernels before it only when they have completed */
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    if (warp < 4) {
        /* 168 registers a thread at launch: 128 * 56 + 256 * 224 = 64512 = 384 * 168 */
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 0) {
            /* -------------------------------------------------------- TMA producer ---- */
            int stage = 0; uint32_t phase = 0;
            uint32_t armed = 0, armed_parity = 0;
            bool alive = true;
            for (int t = cluster_id; t < num_tiles && alive; t += num_clusters) {
                int tm, tn; tile_coords(t, p.tiles_m, p.tiles_n, p.tile_group, tm, tn);
                const int row_a = tm * C::UMMA_M + (int)cta_rank * BM_CTA;
                const int row_b = tn * C::UMMA_N + (int)cta_rank * C::BN;
                for (int kb = 0; kb < p.num_kb; ++kb) {
                    if (!warp_wait(done_bar(stage), phase ^ 1u, p, 1100 + stage, t)) { alive = false; break; }
                    if (elect_one()) {
                        /* both CTAs' bytes are counted on the leader's barrier */
                        if (is_leader) mbar_arrive_expect_tx(full_bar(stage), 2 * C::STAGE_BYTES);
                        const uint32_t fb = mapa(full_bar(stage), 0);
                        if (t != (int)p.waits.lost || kb + 1 < p.num_kb) {
                            tma_load_2d_pair(stage_a(stage), &map_a, fb, kb * BK, row_a);
                            tma_load_2d_pair(stage_b(stage), &map_b, fb, kb * BK, row_b);
                        }
                    }
                    __syncwarp();
                    armed |= 1u << stage;
                    armed_parity = (armed_parity & ~(1u << stage)) | (phase << stage);
                    if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
                }
            }
            /* a wait gave up somewhere: wait (with a limit) for the copies that are still on their way into
             * shared memory; the leader's barriers count its peer's as well, but for a stage that only the peer had filled
             * again, which the peer gives some time */
            if (lane == 0 && gave_up(p.waits)) {
                for (int s2 = 0; is_leader && s2 < C::STAGES; ++s2) {
                    if (!((armed >> s2) & 1u)) continue;
                    for (int tries = 0; tries < 2048 && !mbar_try_wait(full_bar(s2), (armed_parity >> s2) & 1u); ++tries)
                        __nanosleep(64);
                }
                for (int tries = 0; !is_leader && tries < 2048; ++tries) __nanosleep(64);
            }
        } else if (warp == 1) {
            /* -------------------------------------------------------- MMA issuer ------ */
            if (is_leader) {
                int stage = 0; uint32_t phase = 0;
                int unit = 0;                          /* k-blocks so far, over all tiles */
                bool alive = true;
                for (int t = cluster_id; t < num_tiles && alive; t += num_clusters) {
                    for (int kb = 0; kb < p.num_kb; ++kb, ++unit) {
                        const int acc = unit % C::BUFS;
                        if (!warp_wait(full_bar(stage), phase, p, 1300 + stage, t)) { alive = false; break; }
                        if (!warp_wait(tempty_bar(acc), ((uint32_t)(unit / C::BUFS) & 1u) ^ 1u, p, 1200 + acc, t)) { alive = false; break; }
                        tc_fence_after();
                        umma_block<C::CTAS>(tmem_base + (uint32_t)(acc * C::UMMA_N), make_smem_desc(stage_a(stage)), make_smem_desc(stage_b(stage)), p.idesc, done_bar(stage));
                        if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
                    }
                }
                if (!alive && unit > 0) drain_mma(done_bar(stage ? stage - 1 : C::STAGES - 1), stage ? phase : phase ^ 1u);
            }
        } else if (warp == 2) {
            /* -------------------------------------------------------- scale loader ---- */
            constexpr int NA = BM_CTA / 32, NB = COLVEC ? C::UMMA_N / 32 : 1;
            int slot = 0; uint32_t phase = 0;
            bool alive = true;
            for (int t = cluster_id; t < num_tiles && alive; t += num_clusters) {
                int tm, tn; tile_coords(t, p.tiles_m, p.tiles_n, p.tile_group, tm, tn);
                /* this lane's scales of one k-block: rows (columns) lane, lane + 32, ...; without COLVEC lane h < 2 has
                 * the one of the block of column half h */
                const float* src[NA + NB];
                uint32_t exists = 0;
#pragma unroll
                for (int i = 0; i < NA + NB; ++i) {
                    const bool row = i < NA;
                    int64_t r = row ? (int64_t)tm * C::UMMA_M + cta_rank * BM_CTA + i * 32 + lane
                                    : (int64_t)tn * C::UMMA_N + (COLVEC ? (i - NA) * 32 + lane : lane * C::ACC);
                    if (r < (row ? p.M : p.N) && (row || COLVEC || lane < 2)) exists |= 1u << i; else r = 0;
                    src[i] = row ? p.sa.p + (r >> p.sa.shift) * p.sa.rs : p.sb.p + (r >> p.sb.shift) * p.sb.rs;
                }
                for (int kb = 0; kb < p.num_kb; ++kb) {
                    if (!warp_wait(sempty_bar(slot), phase ^ 1u, p, 1500 + slot, t)) { alive = false; break; }
                    const uint32_t dst = ring + (uint32_t)(slot * C::KB_FLOATS + lane) * 4u;
#pragma unroll
                    for (int i = 0; i < NA + NB; ++i) {
                        cp_async4(dst + i * 128u, src[i], (exists >> i) & 1u);
                        src[i] += i < NA ? p.sa.ks : p.sb.ks;
                    }
                    cp_async_arrive(sfull_bar(slot));
                    if (++slot == SLOTS) { slot = 0; phase ^= 1u; }
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        }
    } else {
        /* ------------------------------------------------------------ epilogue -------- */
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        const int q = warp & 3, eh = (warp - 4) >> 2;
        const uint32_t tlane = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(eh * C::ACC);
        const uint32_t box0 = boxes + (uint32_t)(warp - 4) * (4096u * C::BOXES);
        const int box_cols = p.d_type == DECXB_F32 ? 32 : 64;
        uint32_t cphase = 0;                          /* parity of each box's addend */
        uint32_t turn = 0;                            /* boxes stored so far */
        uint32_t pending = 0;                         /* boxes with an addend on its way */
        /* the addend of box i of the tile, once the copy engine has read the results that the box held */
        auto fetch_addend = [&](int i, int64_t col, int64_t row) {
            tma_store_wait_read<0>();
            const uint32_t bar = addend_bar((warp - 4) * 2 + (i & 1));
            mbar_arrive_expect_tx(bar, 4096);
            tma_load_2d(box0 + (uint32_t)(i & 1) * 4096u, &map_c, bar, (int)col, (int)row);
        };
        const uint32_t tempty_at = mapa(tempty_bar(0), 0);      /* the leader's */
        int unit = 0, slot = 0, stage = 0;
        uint32_t sphase = 0, phase = 0;
        bool alive = true;
        for (int t = cluster_id; t < num_tiles && alive; t += num_clusters) {
            int tm, tn; tile_coords(t, p.tiles_m, p.tiles_n, p.tile_group, tm, tn);
            const int64_t row0 = (int64_t)tm * C::UMMA_M + cta_rank * BM_CTA + q * 32;
            const int64_t col0 = (int64_t)tn * C::UMMA_N + eh * C::ACC;
            if (ADDEND && row0 < p.M) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (col0 + i * box_cols < p.N) {
                        if (lane == 0) fetch_addend(i, col0 + i * box_cols, row0);
                        pending |= 1u << i;
                    }
            }
            float sum[C::ACC];
#pragma unroll
            for (int c = 0; c < C::ACC; ++c) sum[c] = 0.0f;
            for (int kb = 0; kb < p.num_kb; ++kb, ++unit) {
                const int acc = unit % C::BUFS;
                if (!warp_wait(sfull_bar(slot), sphase, p, 1600 + slot, t)) { alive = false; break; }
                const uint32_t sc = ring + (uint32_t)(slot * C::KB_FLOATS) * 4u;
                /* this thread's rows: one, or with a factor per column the four of the 16x256b shape */
                float sr[COLVEC ? 4 : 1];
                if constexpr (COLVEC) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) sr[i] = lds_f32(sc + (uint32_t)(q * 32 + i * 8 + (lane >> 2)) * 4u);
                } else {
                    sr[0] = lds_f32(sc + (uint32_t)(q * 32 + lane) * 4u) * lds_f32(sc + (uint32_t)(BM_CTA + eh) * 4u);
                }
                if (!warp_wait(done_bar(stage), phase, p, 1400 + stage, t)) { alive = false; break; }
                tc_fence_after();
                /* 32 columns are multiplied while the next 32 are on their way */
                float v[2][32];
                const uint32_t tacc = tlane + (uint32_t)(acc * C::UMMA_N);
                auto load32 = [&](int c, float* w) {
                    if constexpr (COLVEC) {
                        tmem_ld_16x256<4>(tacc + (uint32_t)c, w);
                        tmem_ld_16x256<4>(tacc + (16u << 16) + (uint32_t)c, w + 16);
                    } else tmem_ld_32x32(tacc + (uint32_t)c, w);
                };
                load32(0, v[0]);
#pragma unroll
                for (int c = 0; c < C::ACC; c += 32) {
                    float* w = v[(c >> 5) & 1];
                    tmem_ld_wait_n<32>(w);
                    if (c + 32 < C::ACC) load32(c + 32, v[((c >> 5) + 1) & 1]);
                    if constexpr (COLVEC) {
                        /* (two numbers an instruction save 8 % of 4096 x 4096 x 8192) */
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            const uint64_t x = lds_b64(sc + (uint32_t)(BM_CTA + eh * C::ACC + c + g * 8 + (lane & 3) * 2) * 4u);
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const int j = (i >> 1) * 16 + g * 4 + (i & 1) * 2;
                                unpack2(fma2(pack2(w[j], w[j + 1]), mul2(pack2(sr[i], sr[i]), x), pack2(sum[c + j], sum[c + j + 1])), sum[c + j], sum[c + j + 1]);
                            }
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; ++j) sum[c + j] = fmaf(w[j], sr[0], sum[c + j]);
                    }
                }
                /* block taken: hand the buffer (in the leader CTA) and the scales' slot back */
                tc_fence_before();
                __syncwarp();
                mbar_arrive_both(tempty_at + 8u * (uint32_t)acc, sempty_bar(slot));
                if (++slot == SLOTS) { slot = 0; sphase ^= 1u; }
                if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
            }
            if (!alive) break;
            if (row0 >= p.M) continue;
#pragma unroll
            for (int c = 0; c < C::ACC; c += 32) {
                if (col0 + c >= p.N) break;
                const float* v = sum + c;
                const bool narrow = p.d_type != DECXB_F32;        /* 64 columns fill a box */
                if (p.tma_store) {
                    const int first = narrow && (c & 32) ? 4 : 0, i = narrow ? c >> 6 : c >> 5;
                    const uint32_t box = box0 + (uint32_t)((ADDEND ? i : (int)turn) & 1) * 4096u;
                    if (first == 0) {
                        if constexpr (ADDEND) {
                            if (!warp_wait(addend_bar((warp - 4) * 2 + (i & 1)), (cphase >> (i & 1)) & 1u, p, 1700 + warp, t)) { alive = false; break; }
                            cphase ^= 1u << (i & 1);
                            pending &= ~(1u << (i & 1));
                        } else {
                            if (lane == 0) tma_store_wait_read<1>();      /* what this box held has been read */
                            __syncwarp();
                        }
                    }
                    box_write<COLVEC, ADDEND>(p.d_type, box, lane, first, v);
                    if (!narrow || first || col0 + c + 32 >= p.N) {
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            tma_store_2d(&map_d, box, (int)(col0 + (narrow ? (c & ~63) : c)), (int)row0);
                            tma_store_commit();
                        }
                        ++turn;
                        /* (only fp32 results have more than two boxes) */
                        if (ADDEND && (i + 2) * box_cols < C::ACC && col0 + (i + 2) * box_cols < p.N) {
                            if (lane == 0) fetch_addend(i + 2, col0 + (i + 2) * box_cols, row0);
                            pending |= 1u << (i & 1);
                        }
                    }
                } else {
                    __syncwarp();
                    box_write<COLVEC, false>(DECXB_F32, box0, lane, 0, v);
                    __syncwarp();
                    if (!narrow)                        box_rows<float>(p, box0, lane, row0, col0 + c + lane);
                    else if (p.d_type == DECXB_F16)     box_rows<__half>(p, box0, lane, row0, col0 + c + lane);
                    else                                box_rows<__nv_bfloat16>(p, box0, lane, row0, col0 + c + lane);
                }
            }
        }
        if (ADDEND && lane == 0)                                  /* a wait gave up: addends may still be on their way */
            for (int i = 0; i < 2; ++i)
                if ((pending >> i) & 1u)
                    for (int tries = 0; tries < 2048 && !mbar_try_wait(addend_bar((warp - 4) * 2 + i), (cphase >> i) & 1u); ++tries) __nanosleep(64);
        if (p.tma_store && lane == 0) tma_store_wait_all();       /* the box stays until the copy engine is done */
    }

    /* ---------------------------------------------------------------- teardown -------- */
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc<C::CTAS>(tmem_base, C::TMEM_COLS);
    }
}

/* --------------------------------------------------------------------------------------
 * Few result tiles: the same product with the roles of the operands exchanged and K split over a cluster.
 *
 * A tile is 128 rows of B (the accumulator's lanes) by NT rows of A (its columns, 16 to 128 tokens), so one token
 * pads the tensor core's tile to 16 columns instead of 128 rows; the CTAs of a cluster take a share of the
 * k-blocks each, and their fp32 sums meet through distributed shared memory: no workspace, no atomics, one order.
 * Bound by the weights' bytes for few tokens (a k-block brings 16 KiB of B whatever NT is): 1 x 8192 x 8192 4.4 TB/s,
 * 64 x 16384 x 16384 5.7 TB/s; below some 30 MB by a launch's 2.4 us and the length of one pass through the pipeline
 * (1 x 4096 x 4096: 5.3 us).
 * Tensor memory is read in the shape in which a thread holds two adjacent columns of every eight for four rows
 * (16x256b), so that a warp's column factors come in a quarter of the shared-memory reads of one row a thread.
 * ------------------------------------------------------------------------------------ */
template <int NT>
struct SplitCfg {
    static constexpr int CTAS_PER_SM = NT == 128 ? 1 : 2;      /* at most, when the launch asks for half of the shared memory (no clusters then) */
    static constexpr int CW = NT / 2;                          /* columns per epilogue warp */
    static constexpr int W_BYTES = BM_CTA * BK;
    static constexpr int STAGE_BYTES = W_BYTES + NT * BK;
    static constexpr int KB_FLOATS = BM_CTA + NT;
    static constexpr int SCALE_BYTES = SLOTS * KB_FLOATS * 4;
    static constexpr int PITCH = BM_CTA + 4;                   /* of the partial sums [NT][PITCH]: no bank twice in a store */
    static constexpr int OTHER_BYTES = SCALE_BYTES + 1024 /* alignment slack */ + 512 /* barriers */;
    static constexpr int MOST_STAGES = 12;
    /* stages of a launch with one or two CTAs per SM */
    static constexpr int stages(int ctas_per_sm)
    {
        const int n = ((ctas_per_sm == 2 ? 113 * 1024 : SMEM_LIMIT) - OTHER_BYTES) / STAGE_BYTES;
        return n > MOST_STAGES ? MOST_STAGES : n;
    }
    static constexpr int BUFS = stages(CTAS_PER_SM) > 4 ? 4 : stages(CTAS_PER_SM) - 1;   /* fewer than stages: their barriers are read by parity */
    static constexpr int TMEM_COLS = 4 * NT;
    static_assert(BUFS >= 2, "buffers");
    static_assert(NT * PITCH * 4 <= stages(CTAS_PER_SM) * STAGE_BYTES, "partial sums reuse the stages");
};

template <int NT>
__global__ void __launch_bounds__(THREADS, SplitCfg<NT>::CTAS_PER_SM)
decxb_gemm_fp8_split_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Params p, const int splits, const int stages)
{
    using C = SplitCfg<NT>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t ring = smem_base + stages * C::STAGE_BYTES;
    const uint32_t bars = ring + C::SCALE_BYTES;
    auto full_bar   = [&](int s) { return bars + 8u * s; };
    auto done_bar   = [&](int s) { return bars + 8u * (C::MOST_STAGES + s); };
    auto tempty_bar = [&](int b) { return bars + 8u * (2 * C::MOST_STAGES + b); };
    auto sfull_bar  = [&](int s) { return bars + 8u * (2 * C::MOST_STAGES + C::BUFS + s); };
    auto sempty_bar = [&](int s) { return bars + 8u * (2 * C::MOST_STAGES + C::BUFS + SLOTS + s); };
    const uint32_t tmem_slot = bars + 8u * (2 * C::MOST_STAGES + C::BUFS + 2 * SLOTS);
    const uint32_t lost = tmem_slot + 4;                                    /* this CTA did not get all of its sums */
    auto stage_w = [&](int s) { return smem_base + s * C::STAGE_BYTES; };
    auto stage_x = [&](int s) { return smem_base + s * C::STAGE_BYTES + C::W_BYTES; };

    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int tile = (int)blockIdx.x / splits, rank = (int)blockIdx.x % splits;
    const int tn = tile / p.tiles_m, tm = tile - tn * p.tiles_m;            /* tokens fastest: their tiles share the weights in L2 */
    const int n0 = tn * BM_CTA, m0 = tm * NT;
    const int kb_first = (int)((int64_t)p.num_kb * rank / splits), kb_last = (int)((int64_t)p.num_kb * (rank + 1) / splits);

    if (threadIdx.x == 0) {
        prefetch_tensormap(&map_w); prefetch_tensormap(&map_x);
        for (int s = 0; s < stages; ++s) { mbar_init(full_bar(s), 1); mbar_init(done_bar(s), 1); }
        for (int b = 0; b < C::BUFS; ++b) mbar_init(tempty_bar(b), EPI_WARPS);
        for (int s = 0; s < SLOTS; ++s) { mbar_init(sfull_bar(s), 32); mbar_init(sempty_bar(s), EPI_WARPS); }
        fence_barrier_init();
        sts_u32(lost, 0);
    }
    if (warp == 1) {
        tmem_alloc<1>(tmem_slot, C::TMEM_COLS);
        tmem_relinquish<1>();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    uint32_t tmem_base;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot));
    /* the next kernel of the stream may take this one's place as its blocks leave; this one starts on the memory of
     * the kernels before it only when they have completed */
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    if (warp == 0) {
        /* ------------------------------------------------------------ TMA producer ---- */
        const int lost_kb = tile == (int)p.waits.lost && rank == 0 ? kb_last - 1 : -1;
        int stage = 0; uint32_t phase = 0;
        uint32_t armed = 0, armed_parity = 0;
        for (int kb = kb_first; kb < kb_last; ++kb) {
            if (!warp_wait(done_bar(stage), phase ^ 1u, p, 2100 + stage, tile)) break;
            if (elect_one()) {
                const uint32_t fb = full_bar(stage);
                mbar_arrive_expect_tx(fb, C::STAGE_BYTES);
                if (kb != lost_kb) {
                    tma_load_2d(stage_w(stage), &map_w, fb, kb * BK, n0);
                    tma_load_2d(stage_x(stage), &map_x, fb, kb * BK, m0);
                }
            }
            __syncwarp();
            armed |= 1u << stage;
            armed_parity = (armed_parity & ~(1u << stage)) | (phase << stage);
            if (++stage == stages) { stage = 0; phase ^= 1u; }
        }
        if (lane == 0 && gave_up(p.waits)) {       /* copies still on their way */
            for (int s2 = 0; s2 < stages; ++s2) {
                if (!((armed >> s2) & 1u)) continue;
                for (int tries = 0; tries < 2048 && !mbar_try_wait(full_bar(s2), (armed_parity >> s2) & 1u); ++tries) __nanosleep(64);
            }
        }
    } else if (warp == 1) {
        /* ------------------------------------------------------------ MMA issuer ------ */
        int stage = 0; uint32_t phase = 0;
        for (int unit = 0; unit < kb_last - kb_first; ++unit) {
            const int acc = unit % C::BUFS;
            if (!warp_wait(full_bar(stage), phase, p, 2300 + stage, tile) ||
                !warp_wait(tempty_bar(acc), ((uint32_t)(unit / C::BUFS) & 1u) ^ 1u, p, 2200 + acc, tile)) {
                if (unit > 0) drain_mma(done_bar(stage ? stage - 1 : stages - 1), stage ? phase : phase ^ 1u);
                break;
            }
            tc_fence_after();
            umma_block<1>(tmem_base + (uint32_t)(acc * NT), make_smem_desc(stage_w(stage)), make_smem_desc(stage_x(stage)), p.idesc, done_bar(stage));
            if (++stage == stages) { stage = 0; phase ^= 1u; }
        }
    } else if (warp == 2) {
        /* ------------------------------------------------------------ scale loader ---- */
        constexpr int NX = (NT + 31) / 32;
        const float* src[4 + NX];
        uint32_t exists = 0;
#pragma unroll
        for (int i = 0; i < 4 + NX; ++i) {
            const bool w = i < 4;
            const int at = (w ? i : i - 4) * 32 + lane;
            int64_t r = (int64_t)(w ? n0 : m0) + at;
            if (r < (w ? p.N : p.M) && (w || at < NT)) exists |= 1u << i; else r = 0;
            src[i] = w ? p.sb.p + (r >> p.sb.shift) * p.sb.rs + kb_first * p.sb.ks : p.sa.p + (r >> p.sa.shift) * p.sa.rs + kb_first * p.sa.ks;
        }
        int slot = 0; uint32_t phase = 0;
        for (int kb = kb_first; kb < kb_last; ++kb) {
            if (!warp_wait(sempty_bar(slot), phase ^ 1u, p, 2500 + slot, tile)) break;
            const uint32_t dst = ring + (uint32_t)(slot * C::KB_FLOATS + lane) * 4u;
#pragma unroll
            for (int i = 0; i < 4 + NX; ++i) {
                if (i < 4 || NT >= 32 || lane < NT) cp_async4(dst + i * 128u, src[i], (exists >> i) & 1u);
                src[i] += i < 4 ? p.sb.ks : p.sa.ks;
            }
            cp_async_arrive(sfull_bar(slot));
            if (++slot == SLOTS) { slot = 0; phase ^= 1u; }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp >= 4) {
        /* ------------------------------------------------------------ sums ------------ */
        const int q = warp & 3, eh = (warp - 4) >> 2;
        constexpr int G = C::CW >= 32 ? 4 : C::CW / 8;         /* groups of eight columns per load */
        const uint32_t tlane = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(eh * C::CW);
        float sum[C::CW];                                      /* [columns / 8 G][lane half][G][4] */
#pragma unroll
        for (int i = 0; i < C::CW; ++i) sum[i] = 0.0f;
        int stage = 0, slot = 0;
        uint32_t phase = 0, sphase = 0;
        bool alive = true;
        for (int unit = 0; unit < kb_last - kb_first; ++unit) {
            const int acc = unit % C::BUFS;
            if (!warp_wait(sfull_bar(slot), sphase, p, 2600 + slot, tile)) { alive = false; break; }
            const uint32_t sc = ring + (uint32_t)(slot * C::KB_FLOATS) * 4u;
            float sw[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) sw[i] = lds_f32(sc + (uint32_t)(q * 32 + i * 8 + (lane >> 2)) * 4u);
            if (!warp_wait(done_bar(stage), phase, p, 2400 + stage, tile)) { alive = false; break; }
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < C::CW; c += 8 * G) {
                float v[8 * G];
                tmem_ld_16x256<G>(tlane + (uint32_t)(acc * NT + c), v);
                tmem_ld_16x256<G>(tlane + (16u << 16) + (uint32_t)(acc * NT + c), v + 4 * G);
                tmem_ld_wait_n<8 * G>(v);
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const float2 x = lds_f32x2(sc + (uint32_t)(BM_CTA + eh * C::CW + c + g * 8 + (lane & 3) * 2) * 4u);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int i = h * 4 * G + g * 4 + k;
                            sum[c + i] = fmaf(v[i], sw[2 * h + (k >> 1)] * ((k & 1) ? x.y : x.x), sum[c + i]);
                        }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (elect_one()) { mbar_arrive(tempty_bar(acc)); mbar_arrive(sempty_bar(slot)); }
            __syncwarp();
            if (++slot == SLOTS) { slot = 0; sphase ^= 1u; }
            if (++stage == stages) { stage = 0; phase ^= 1u; }
        }
        if (alive) {
            /* every MMA of this CTA has run, so the stages can hold its sums: [token][row of B] */
#pragma unroll
            for (int c = 0; c < C::CW; c += 8 * G)
#pragma unroll
                for (int i = 0; i < 8 * G; ++i) {
                    const int h = i / (4 * G), g = (i / 4) % G, k = i & 3;
                    const int m = eh * C::CW + c + g * 8 + (lane & 3) * 2 + (k & 1), n = q * 32 + h * 16 + (k >> 1) * 8 + (lane >> 2);
                    asm volatile("st.shared.f32 [%0], %1;" :: "r"(smem_base + (uint32_t)(m * C::PITCH + n) * 4u), "f"(sum[c + i]) : "memory");
                }
        } else {
            /* a wait gave up: NaN in place of this warp's sums, which makes those who add them ask, once the copies that are still
             * on their way into the stages have had their time */
            for (int tries = 0; tries < 2048; ++tries) __nanosleep(64);
            for (int m = eh * C::CW; m < (eh + 1) * C::CW; ++m) sts_u32(smem_base + (uint32_t)(m * C::PITCH + q * 32 + lane) * 4u, 0x7fffffffu);
            if (lane == 0) sts_u32(lost, 1);
        }
    }
    __syncwarp();
    tc_fence_before();
    if (splits > 1) cluster_sync_all(); else __syncthreads();

    /* each CTA finishes its share of the tokens, eight at a time, four columns a thread: the cluster's sums in ascending
     * order, addend, one rounding.  Where a CTA did not get its sums, D stays as it was; the peers' words on that are read only where a
     * sum is NaN (asked for every tile they cost 1 to 4 %) */
    if (warp >= 4) {
        const int t = (int)threadIdx.x - 128, n = n0 + (t & 31) * 4, rows = (int)min((int64_t)NT, p.M - m0);
        const int have = (int)min((int64_t)4, p.N - n);
        for (int m = rank * 8 + (t >> 5); m < rows && have > 0; m += 8 * splits) {
            const uint32_t at = smem_base + (uint32_t)(m * C::PITCH + (t & 31) * 4) * 4u;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
            for (int r = 0; r < splits; ++r) {
                const float4 w = splits > 1 ? lds_cluster_f32x4(mapa(at, (uint32_t)r)) : lds_f32x4(at);
                v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
            }
            if (v.x != v.x) {
                bool gone = false;
#pragma unroll 1
                for (int r = 0; r < splits; ++r) gone |= lds_cluster_u32(mapa(lost, (uint32_t)r)) != 0;
                if (gone) continue;
            }
            if (p.d_type == DECXB_F32)      put4<float>(p, m0 + m, n, have, v);
            else if (p.d_type == DECXB_F16) put4<__half>(p, m0 + m, n, have, v);
            else                            put4<__nv_bfloat16>(p, m0 + m, n, have, v);
        }
    }
    __syncwarp();
    if (splits > 1) cluster_sync_all(); else __syncthreads();      /* the peers have read this CTA's sums */
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc<1>(tmem_base, C::TMEM_COLS);
    }
}

/* ------------------------------------------------------------------ host side -------- */
/* rows x cols array of 1-, 2- or 4-byte elements with a row pitch of `ld` elements; box = 128 bytes x box_rows, 128-byte swizzle. */
int make_map_2d(decxb_ctx* ctx, CUtensorMap* map, CUtensorMapDataType type, int e, const void* base, int64_t rows, int64_t cols,
                int64_t ld, int box_rows)
{
    auto fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(decxb_tensor_map_encoder());
    if (!fn) return decxb_fail(ctx, DECXB_ERR_CUDA, "cuTensorMapEncodeTiled entry point not found");
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)(ld * e)};
    cuuint32_t box[2] = {(cuuint32_t)(128 / e), (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(map, type, 2, const_cast<void*>(base), dims, strides, box, estr,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return decxb_fail(ctx, DECXB_ERR_CUDA, "cuTensorMapEncodeTiled (fp8) failed: " + std::to_string((int)r));
    return DECXB_OK;
}

int make_map_fp8(decxb_ctx* ctx, CUtensorMap* map, const decxb_fp8_matrix& m, int box_rows)
{
    return make_map_2d(ctx, map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, m.data, m.rows, m.cols, m.ld, box_rows);
}

template <bool COLVEC, bool ADDEND>
int launch(decxb_ctx* ctx, const decxb_fp8_matrix& A, const decxb_fp8_matrix& B, Params p, cudaStream_t s)
{
    using C = Cfg<COLVEC>;
    auto kernel = decxb_gemm_fp8_kernel<COLVEC, ADDEND>;
    static std::once_flag once[DECXB_MAX_DEVICES];
    static cudaError_t attr_err[DECXB_MAX_DEVICES];
    static int regs[DECXB_MAX_DEVICES];
    const int dev = ctx->device;
    std::call_once(once[dev], [&] {
        attr_err[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES);
        cudaFuncAttributes fa;
        if (attr_err[dev] == cudaSuccess) attr_err[dev] = cudaFuncGetAttributes(&fa, kernel);
        if (attr_err[dev] == cudaSuccess) regs[dev] = fa.numRegs;
    });
    if (attr_err[dev] != cudaSuccess) return decxb_fail(ctx, DECXB_ERR_CUDA, std::string("fp8 kernel attributes: ") + cudaGetErrorString(attr_err[dev]));
    /* a register hand-over that does not add up would wait forever: never launch it */
    if (regs[dev] != 168) return decxb_fail(ctx, DECXB_ERR_CUDA, "fp8 GEMM kernel was not compiled to 168 registers");
    CUtensorMap ma, mb;
    int rc;
    if ((rc = make_map_fp8(ctx, &ma, A, BM_CTA)) || (rc = make_map_fp8(ctx, &mb, B, C::BN))) return rc;
    CUtensorMap md = ma, mc = ma;
    if (p.tma_store) {
        const int e = size_of(p.d_type);
        const CUtensorMapDataType type = p.d_type == DECXB_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                       : p.d_type == DECXB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
        if ((rc = make_map_2d(ctx, &md, type, e, p.D, p.M, p.N, p.ldd, 32))) return rc;
        if (ADDEND && (rc = make_map_2d(ctx, &mc, type, e, p.C, p.M, p.N, p.ldc, 32))) return rc;
    }
    const int64_t tm = decxb_ceil_div(p.M, C::UMMA_M), tn = decxb_ceil_div(p.N, C::UMMA_N);
    if (tm * tn > 0x7fffffffLL) return decxb_fail(ctx, DECXB_ERR_TOO_LARGE, "fp8 gemm tiles");
    p.tiles_m = (int)tm; p.tiles_n = (int)tn;
    p.idesc = make_idesc_fp8(C::UMMA_M, C::UMMA_N, A.type, B.type);
    int64_t clusters = (ctx->sm_count - ctx->reserved_sms) / C::CTAS;
    if (clusters > tm * tn) clusters = tm * tn;
    if (clusters < 1) clusters = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(clusters * C::CTAS), 1, 1);
    cfg.blockDim = dim3(THREADS, 1, 1);
    cfg.dynamicSmemBytes = C::SMEM_BYTES;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C::CTAS; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    decxb_launch_scope scope(ctx, s, DECXB_K_GEMM);
    DECXB_CUDA_TRY(ctx, cudaLaunchKernelEx(&cfg, kernel, ma, mb, md, mc, p));
    return DECXB_OK;
}

/* The launch of a split product but for its stream: `clusters` clusters of `splits` CTAs, `per_sm` CTAs to an SM. */
template <int NT>
cudaLaunchConfig_t split_config(cudaLaunchAttribute* attr, int64_t clusters, int splits, int per_sm)
{
    using C = SplitCfg<NT>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(clusters * splits), 1, 1);
    cfg.blockDim = dim3(THREADS, 1, 1);
    cfg.dynamicSmemBytes = (size_t)C::stages(per_sm) * C::STAGE_BYTES + C::OTHER_BYTES;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)splits; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    return cfg;
}

/* How many clusters of 1, 2, 4 and 8 CTAs the device holds at once with one CTA to an SM (asked once): the SMs of a cluster lie
 * in one group of SMs, so it is less than the SMs divided by the size. */
struct Resident { int clusters[4]; cudaError_t err; };

template <int NT>
const Resident& resident(decxb_ctx* ctx)
{
    static std::once_flag once[DECXB_MAX_DEVICES];
    static Resident table[DECXB_MAX_DEVICES];
    Resident& t = table[ctx->device];
    std::call_once(once[ctx->device], [&] {
        auto kernel = decxb_gemm_fp8_split_kernel<NT>;
        t.err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_LIMIT);
        for (int i = 0; i < 4 && t.err == cudaSuccess; ++i) {
            cudaLaunchAttribute attr[2];
            cudaLaunchConfig_t cfg = split_config<NT>(attr, 1, 1 << i, 1);
            cfg.numAttrs = 1;
            t.err = cudaOccupancyMaxActiveClusters(&t.clusters[i], kernel, &cfg);
        }
    });
    return t;
}

/* How a product is cut: `splits` shares of K, `per_sm` CTAs to an SM (two have half the stages each), and what it takes, in
 * microseconds (fitted to 65 <= M <= 1024, 1024 <= N <= 32768, 1024 <= K <= 16384 on a B200).
 *  - The largest power of two of shares of which one wave of clusters holds all (2048 columns, K = 4096, one token: 2, 4, 8
 *    shares 6.6, 4.7, 8.2 us, eight being two waves), but no share below four k-blocks (1 x 4096 x 1024: two shares
 *    3.9, four 4.3, eight 5.2 us).
 *  - Up to 64 tokens, two CTAs to an SM where there are more tiles than SMs (64 x 32768 x 4096: 32.3 and 26.4). Otherwise one CTA
 *    with all of the shared memory has the longer queue of loads (48 x 4096 x 8192: 10.3 and 14.6).
 *  - Never a cluster of CTAs that leave room on their SMs: tensor memory is taken in the order in which blocks come, without
 *    a limit to the wait, and a CTA that holds some while it waits for its peer, next to a block of another kernel that does the same
 *    the other way round, would wait for good.  (Twice the shares with two CTAs to an SM, where a fifth of the SMs are
 *    empty: 1 x 6000 x 4096 6.97 -> 6.56 us, 40 x 5000 x 4096 9.4 -> 10.1.) */
struct Cut { int splits, per_sm; double us; };

template <int NT>
int plan_split(decxb_ctx* ctx, int64_t M, int64_t N, int num_kb, Cut* out)
{
    const Resident& r = resident<NT>(ctx);
    if (r.err != cudaSuccess) return decxb_fail(ctx, DECXB_ERR_CUDA, std::string("fp8 kernel attributes: ") + cudaGetErrorString(r.err));
    const int64_t tiles = decxb_ceil_div(M, NT) * decxb_ceil_div(N, BM_CTA);
    int i = 3;
    while (i > 0 && (tiles > r.clusters[i] || num_kb < (4 << i))) --i;
    Cut c = {1 << i, 1, 0.0};
    const int fit = r.clusters[i] > 0 ? r.clusters[i] : 1;
    const int64_t waves = decxb_ceil_div(tiles, fit);
    c.us = 5.0 + (waves > 1 ? 0.50 : 0.36) * (double)waves * (double)decxb_ceil_div(num_kb, c.splits);
    if (SplitCfg<NT>::CTAS_PER_SM == 2 && tiles > fit) c.per_sm = 2;
    *out = c;
    return DECXB_OK;
}

template <int NT>
int launch_split(decxb_ctx* ctx, const decxb_fp8_matrix& A, const decxb_fp8_matrix& B, Params p, const Cut& cut, cudaStream_t s)
{
    using C = SplitCfg<NT>;
    CUtensorMap mw, mx;
    int rc;
    if ((rc = make_map_fp8(ctx, &mw, B, BM_CTA)) || (rc = make_map_fp8(ctx, &mx, A, NT))) return rc;
    const int64_t tm = decxb_ceil_div(p.M, NT), tn = decxb_ceil_div(p.N, BM_CTA);
    if (tm * tn * cut.splits > 0x7fffffffLL) return decxb_fail(ctx, DECXB_ERR_TOO_LARGE, "fp8 gemm tiles");
    p.tiles_m = (int)tm; p.tiles_n = (int)tn;
    p.idesc = make_idesc_fp8(BM_CTA, NT, B.type, A.type);
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg = split_config<NT>(attr, tm * tn, cut.splits, cut.per_sm);
    cfg.stream = s;
    decxb_launch_scope scope(ctx, s, DECXB_K_GEMM);
    DECXB_CUDA_TRY(ctx, cudaLaunchKernelEx(&cfg, decxb_gemm_fp8_split_kernel<NT>, mw, mx, p, cut.splits, C::stages(cut.per_sm)));
    return DECXB_OK;
}

template <int NT>
int plan_and_launch_split(decxb_ctx* ctx, const decxb_fp8_matrix& A, const decxb_fp8_matrix& B, const Params& p, cudaStream_t s)
{
    Cut cut;
    const int rc = plan_split<NT>(ctx, p.M, p.N, p.num_kb, &cut);
    return rc ? rc : launch_split<NT>(ctx, A, B, p, cut, s);
}

/* The kernel of a product: tiles of NT tokens for up to 64 tokens, otherwise what takes less, split tiles of 128 tokens or
 * pairs' tiles of 256 x 256 (512 x 4096 x 4096: 19.1 and 18.7 us; 256 x 4096 x 4096: 13.6 and 18.3). */
int launch_product(decxb_ctx* ctx, const decxb_fp8_matrix& A, const decxb_fp8_matrix& B, const Params& p, cudaStream_t s)
{
    if (p.M <= 16) return plan_and_launch_split<16>(ctx, A, B, p, s);
    if (p.M <= 32) return plan_and_launch_split<32>(ctx, A, B, p, s);
    if (p.M <= 64) return plan_and_launch_split<64>(ctx, A, B, p, s);
    Cut cut;
    if (int rc = plan_split<128>(ctx, p.M, p.N, p.num_kb, &cut)) return rc;
    const bool by_row = B.block_rows == 1;
    const int64_t pairs = decxb_ceil_div(p.M, 256) * decxb_ceil_div(p.N, 256), at_once = ctx->sm_count / 2 > 0 ? ctx->sm_count / 2 : 1;
    const double pair_us = 5.0 + (by_row ? 0.80 : 0.42) * (double)decxb_ceil_div(pairs, at_once) * (double)p.num_kb;
    if (cut.us < pair_us) return launch_split<128>(ctx, A, B, p, cut, s);
    if (p.C && p.tma_store) return by_row ? launch<true, true>(ctx, A, B, p, s) : launch<false, true>(ctx, A, B, p, s);
    return by_row ? launch<true, false>(ctx, A, B, p, s) : launch<false, false>(ctx, A, B, p, s);
}

/* Codes that the copy engine cannot address are copied to a pitch it can. */
int reachable(decxb_ctx* ctx, decxb_fp8_matrix* m, void** scratch, cudaStream_t s)
{
    if (m->rows == 1) m->ld = decxb_ceil_to(m->cols, 16);          /* a single row has no pitch */
    if (aligned(m->data, m->ld, 16)) return DECXB_OK;
    int rc;
    if ((rc = refuse_capture(ctx, s, "an operand's address or ld is not a multiple of 16 bytes"))) return rc;
    const int64_t ld = decxb_ceil_to(m->cols, 16);
    if ((rc = decxb_malloc_on_stream(ctx, (size_t)m->rows * ld, scratch, s))) return rc;
    DECXB_CUDA_TRY(ctx, cudaMemcpy2DAsync(*scratch, ld, m->data, m->ld, m->cols, m->rows, cudaMemcpyDeviceToDevice, s));
    m->data = *scratch; m->ld = ld;
    return DECXB_OK;
}

ScaleView view_of(const decxb_fp8_matrix& m)
{
    return {m.scales, m.scale_row_stride, m.scale_block_stride, m.block_rows == 128 ? 7 : 0};
}

int gemm_fp8(decxb_ctx* ctx, const decxb_fp8_matrix* pa, const decxb_fp8_matrix* pb, const void* C, int64_t ldc,
             void* D, int d_type, int64_t ldd, cudaStream_t s)
{
    if (!pa || !pb) return decxb_fail(ctx, DECXB_ERR_BAD_PARAM, "null operand");
    if (!type_ok(d_type)) return decxb_fail(ctx, DECXB_ERR_BAD_FLAG, "d_type");
    int rc;
    if ((rc = check_matrix(ctx, pa, "A", -1, -1)) || (rc = check_matrix(ctx, pb, "B", -1, pa->cols))) return rc;
    if (pa->cols == 0) return decxb_fail(ctx, DECXB_ERR_BAD_PARAM, "K must be positive");
    const int64_t M = pa->rows, N = pb->rows;
    if (M == 0 || N == 0) return DECXB_OK;
    const int e = size_of(d_type);
    if ((rc = check_array(ctx, D, ldd, N, e, "D"))) return rc;
    if (C && (rc = check_array(ctx, C, ldc, N, e, "C"))) return rc;
    if (C == D && ldc != ldd) return decxb_fail(ctx, DECXB_ERR_BAD_PARAM, "C in place of D needs its leading dimension");
    decxb_fp8_matrix A = *pa, B = *pb;
    void *a_copy = nullptr, *b_copy = nullptr;
    rc = reachable(ctx, &A, &a_copy, s);
    if (rc == DECXB_OK) rc = reachable(ctx, &B, &b_copy, s);
    if (rc == DECXB_OK) {
        Params p = {};
        p.M = M; p.N = N;
        p.num_kb = (int)decxb_ceil_div(A.cols, BK);
        p.tile_group = ctx->tile_group > 0 ? ctx->tile_group : 8;
        p.sa = view_of(A); p.sb = view_of(B);
        p.C = C; p.ldc = ldc; p.D = D; p.ldd = ldd; p.d_type = d_type;
        /* the copy engine clips a store at the array's edge in whole 16-byte pieces, so N has to be made of them too */
        p.tma_store = aligned(D, ldd * e, 16) && (!C || aligned(C, ldc * e, 16)) && N * e % 16 == 0;
        p.d_vec = aligned(D, ldd * e, 4 * e);
        p.waits = waits_of(ctx);
        rc = launch_product(ctx, A, B, p, s);
    }
    if (a_copy) decxb_free_on_stream(ctx, a_copy, s);
    if (b_copy) decxb_free_on_stream(ctx, b_copy, s);
    return rc;
}

}  // namespace

extern "C" int decxb_gemm_fp8(decxb_ctx* ctx, const decxb_fp8_matrix* A, const decxb_fp8_matrix* B,
                              const void* C, int64_t ldc, void* D, int d_type, int64_t ldd, void* stream)
try {
    DeviceScope dev(ctx);
    if (dev.status) return dev.status;
    return gemm_fp8(ctx, A, B, C, ldc, D, d_type, ldd, stream ? (cudaStream_t)stream : ctx->stream);
} catch (...) { return DECXB_ERR_ALLOC; }      /* the host's memory, or a lock of the runtime */
