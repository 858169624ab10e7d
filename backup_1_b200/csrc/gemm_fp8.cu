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
 *  - Warp-specialised, persistent: warp 0 = TMA producer, warp 1 = MMA issuer and tensor-memory owner, warps 2 and 3 =
 *    scale loaders (cp.async into a ring of their own, eight k-blocks ahead), warps 4..11 = epilogue (four lane
 *    quarters x two column halves).
 *  - Every wait on an mbarrier is bounded; on expiry the waiter records where it gave up in the context's status word,
 *    all roles drain and the kernel returns.
 */
#include "fp8.cuh"
#include "tc_ptx.cuh"

#include <cudaTypedefs.h>

#include <mutex>
#include <new>

namespace {

using namespace tcptx;
using namespace fp8;

constexpr int BM_CTA = 128;        /* rows of A (and accumulator lanes) per CTA      */
constexpr int BK = 128;            /* codes per k-block                               */
constexpr int UMMA_K = 32;         /* k per tcgen05.mma kind::f8f6f4                   */
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
    bool d_vec, c_vec;             /* 128-bit accesses to D / C                        */
    long long wait_limit_ns;
    decxb_dev_status* status;
};

/* Bounded wait of one thread; false when it gave up or another role already had. */
__device__ __forceinline__ bool wait_bounded(uint32_t bar, uint32_t parity, const Params& p, int where, int detail)
{
    if (mbar_try_wait(bar, parity)) return true;
    const unsigned long long t0 = globaltimer_ns();
    uint32_t spins = 0;
    while (!mbar_try_wait(bar, parity)) {
        if ((++spins & 1023u) == 0) {
            if (*reinterpret_cast<volatile int*>(&p.status->code) != 0) return false;
            if ((long long)(globaltimer_ns() - t0) > p.wait_limit_ns) {
                if (atomicCAS(&p.status->code, 0, DECXB_DEVERR_WAIT_EXPIRED) == 0) {
                    p.status->where = where; p.status->block = (int)blockIdx.x; p.status->detail = detail;
                    __threadfence_system();
                }
                return false;
            }
        }
    }
    return true;
}

/* The same for a whole warp that goes on together (tcgen05.ld is warp-wide): one lane's giving up is all lanes'. */
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, const Params& p, int where, int detail)
{
    return __all_sync(0xffffffffu, wait_bounded(bar, parity, p, where, detail));
}

template <int CTAS>
__device__ __forceinline__ void umma_fp8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate)
{
    if (CTAS == 1)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                     :: "r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                     :: "r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
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

/* Two fp32 lanes per instruction. */
__device__ __forceinline__ uint64_t pack2(float a, float b)
{
    uint64_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b)
{
    uint64_t r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r;
}

/* Tile order: groups of `group` tile-rows, column by column inside a group (operand panels shared in L2). */
__device__ __forceinline__ void tile_coords(int t, int tiles_m, int tiles_n, int group, int& tm, int& tn)
{
    const int per_group = group * tiles_n, g = t / per_group, first_m = g * group;
    const int gsz = min(tiles_m - first_m, group), r = t - g * per_group;
    tm = first_m + r % gsz;
    tn = r / gsz;
}

/* Eight result columns from `col` on of one row: (+C), one rounding, 128-bit stores where the rows allow them. */
template <typename T>
__device__ __forceinline__ void store_row8(const Params& p, int64_t row, int64_t col, float* v)
{
    const int n = (int)min((int64_t)8, p.N - col);
    if (n <= 0) return;
    if (p.C) {
        float c[8];
        load8(static_cast<const T*>(p.C) + row * p.ldc + col, n, p.c_vec, c);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += c[j];
    }
    store8(static_cast<T*>(p.D) + row * p.ldd + col, n, p.d_vec, v);
}

/* --------------------------------------------------------------------------------------
 * CTAS   : 1 or 2 CTAs per tile (cta_group)
 * BN     : rows of B loaded per CTA; the tile is 128 CTAS x BN CTAS
 * COLVEC : B has a scale per row (block_rows 1): each column of the tile has its own factor.  Otherwise a
 *          128-row block of B has one scale, and the columns of one epilogue warp lie in one block.
 * ------------------------------------------------------------------------------------ */
template <int CTAS, int BN, bool COLVEC>
struct Cfg {
    static constexpr int UMMA_M = BM_CTA * CTAS;
    static constexpr int UMMA_N = BN * CTAS;
    static constexpr int ACC = UMMA_N / 2;                     /* columns per epilogue warp */
    static constexpr int A_BYTES = BM_CTA * BK;
    static constexpr int B_BYTES = BN * BK;
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int SLOT_FLOATS = BM_CTA + (COLVEC ? UMMA_N : 32);
    static constexpr int SCALE_BYTES = SLOTS * SLOT_FLOATS * 4;
    static constexpr int STAGES_RAW = (SMEM_LIMIT - 2048 - SCALE_BYTES) / STAGE_BYTES;
    static constexpr int STAGES = STAGES_RAW > 8 ? 8 : STAGES_RAW;
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + SCALE_BYTES + 1024 /* alignment slack */ + 512 /* barriers */;
    static constexpr int TMEM_COLS = 2 * UMMA_N;               /* two buffers */
    /* 128 running sums per thread need the registers of warp group 0: see the launch */
    static constexpr bool REALLOC = ACC > 64;
    static_assert(UMMA_N % 64 == 0 && UMMA_N <= 256 && ACC <= 128, "tile width");
    static_assert(SMEM_BYTES <= SMEM_LIMIT && STAGES >= 3, "shared memory");
};

template <int CTAS, int BN, bool COLVEC>
__global__ void __launch_bounds__(THREADS, 1)
decxb_gemm_fp8_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Params p)
{
    using C = Cfg<CTAS, BN, COLVEC>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;     /* the swizzle is a function of address bits 4-9 */
    const uint32_t ring = smem_base + C::STAGES * C::STAGE_BYTES;
    const uint32_t bars = ring + C::SCALE_BYTES;
    auto full_bar   = [&](int s) { return bars + 8u * s; };
    auto empty_bar  = [&](int s) { return bars + 8u * (C::STAGES + s); };
    auto tfull_bar  = [&](int b) { return bars + 8u * (2 * C::STAGES + b); };
    auto tempty_bar = [&](int b) { return bars + 8u * (2 * C::STAGES + 2 + b); };
    auto sfull_bar  = [&](int s) { return bars + 8u * (2 * C::STAGES + 4 + s); };
    auto sempty_bar = [&](int s) { return bars + 8u * (2 * C::STAGES + 4 + SLOTS + s); };
    const uint32_t tmem_slot = bars + 8u * (2 * C::STAGES + 4 + 2 * SLOTS);
    auto stage_a = [&](int s) { return smem_base + s * C::STAGE_BYTES; };
    auto stage_b = [&](int s) { return smem_base + s * C::STAGE_BYTES + C::A_BYTES; };

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t cta_rank = CTAS == 2 ? cluster_ctarank() : 0u;
    const bool is_leader = cta_rank == 0;
    const int cluster_id = (int)blockIdx.x / CTAS, num_clusters = (int)gridDim.x / CTAS;
    const int num_tiles = p.tiles_m * p.tiles_n;

    if (threadIdx.x == 0) {
        prefetch_tensormap(&map_a); prefetch_tensormap(&map_b);
        for (int s = 0; s < C::STAGES; ++s) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(tfull_bar(b), 1); mbar_init(tempty_bar(b), EPI_WARPS * CTAS); }
        for (int s = 0; s < SLOTS; ++s) { mbar_init(sfull_bar(s), 64); mbar_init(sempty_bar(s), EPI_WARPS); }
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc<CTAS>(tmem_slot, C::TMEM_COLS);
        tmem_relinquish<CTAS>();
    }
    tc_fence_before();
    __syncthreads();
    if (CTAS == 2) cluster_sync_all();
    tc_fence_after();
    uint32_t tmem_base;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot));
    asm volatile("griddepcontrol.wait;" ::: "memory");

    if (warp < 4) {
        /* 168 registers a thread at launch: 128 * 56 + 256 * 224 = 64512 = 384 * 168 */
        if constexpr (C::REALLOC) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 0) {
            /* -------------------------------------------------------- TMA producer ---- */
            if (lane == 0) {
                int stage = 0; uint32_t phase = 0;
                uint32_t armed = 0, armed_parity = 0;
                bool alive = true;
                for (int t = cluster_id; t < num_tiles && alive; t += num_clusters) {
                    int tm, tn; tile_coords(t, p.tiles_m, p.tiles_n, p.tile_group, tm, tn);
                    const int row_a = tm * C::UMMA_M + (int)cta_rank * BM_CTA;
                    const int row_b = tn * C::UMMA_N + (int)cta_rank * BN;
                    for (int kb = 0; kb < p.num_kb; ++kb) {
                        if (!wait_bounded(empty_bar(stage), phase ^ 1u, p, 1100 + stage, t)) { alive = false; break; }
                        if (CTAS == 1) {
                            const uint32_t fb = full_bar(stage);
                            mbar_arrive_expect_tx(fb, C::STAGE_BYTES);
                            tma_load_2d(stage_a(stage), &map_a, fb, kb * BK, row_a);
                            tma_load_2d(stage_b(stage), &map_b, fb, kb * BK, row_b);
                        } else {
                            /* both CTAs' bytes are counted on the leader's barrier */
                            if (is_leader) mbar_arrive_expect_tx(full_bar(stage), 2 * C::STAGE_BYTES);
                            const uint32_t fb = mapa(full_bar(stage), 0);
                            tma_load_2d_pair(stage_a(stage), &map_a, fb, kb * BK, row_a);
                            tma_load_2d_pair(stage_b(stage), &map_b, fb, kb * BK, row_b);
                        }
                        armed |= 1u << stage;
                        armed_parity = (armed_parity & ~(1u << stage)) | (phase << stage);
                        if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
                    }
                }
                /* a wait gave up somewhere: wait (with a limit) for the copies that are still on their way into
                 * shared memory; the leader's barriers count its peer's as well */
                if (is_leader && *reinterpret_cast<volatile int*>(&p.status->code) != 0) {
                    for (int s2 = 0; s2 < C::STAGES; ++s2) {
                        if (!((armed >> s2) & 1u)) continue;
                        for (int tries = 0; tries < 2048 && !mbar_try_wait(full_bar(s2), (armed_parity >> s2) & 1u); ++tries)
                            __nanosleep(64);
                    }
                }
            }
        } else if (warp == 1) {
            /* -------------------------------------------------------- MMA issuer ------ */
            if (is_leader && lane == 0) {
                int stage = 0; uint32_t phase = 0;
                int unit = 0;                          /* k-blocks so far, over all tiles */
                bool alive = true;
                for (int t = cluster_id; t < num_tiles && alive; t += num_clusters) {
                    for (int kb = 0; kb < p.num_kb; ++kb, ++unit) {
                        const int acc = unit & 1;
                        if (!wait_bounded(tempty_bar(acc), ((uint32_t)(unit >> 1) & 1u) ^ 1u, p, 1200 + acc, t)) { alive = false; break; }
                        if (!wait_bounded(full_bar(stage), phase, p, 1300 + stage, t)) { alive = false; break; }
                        tc_fence_after();
                        const uint32_t tmem_d = tmem_base + (uint32_t)(acc * C::UMMA_N);
                        const uint64_t da = make_smem_desc(stage_a(stage)), db = make_smem_desc(stage_b(stage));
#pragma unroll
                        for (int kk = 0; kk < BK / UMMA_K; ++kk) {
                            const uint64_t koff = (uint64_t)((kk * UMMA_K) >> 4);
                            umma_fp8<CTAS>(tmem_d, da + koff, db + koff, p.idesc, kk != 0 ? 1u : 0u);
                        }
                        umma_commit<CTAS>(empty_bar(stage));     /* stage reusable once these MMAs have read it */
                        umma_commit<CTAS>(tfull_bar(acc));       /* k-block summed */
                        if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
                    }
                }
            }
        } else {
            /* -------------------------------------------------------- scale loaders --- */
            const bool rows = warp == 2;
            constexpr int NA = BM_CTA / 32, NB = COLVEC ? C::UMMA_N / 32 : 1;
            int slot = 0; uint32_t phase = 0;
            bool alive = true;
            for (int t = cluster_id; t < num_tiles && alive; t += num_clusters) {
                int tm, tn; tile_coords(t, p.tiles_m, p.tiles_n, p.tile_group, tm, tn);
                /* this lane's scales of one k-block: rows (columns) lane, lane + 32, ...; without COLVEC lane h < 2 has
                 * the one of the block of column half h */
                constexpr int NMOST = NA > NB ? NA : NB;
                const float* src[NMOST];
                uint32_t exists = 0;
#pragma unroll
                for (int i = 0; i < NMOST; ++i) {
                    int64_t r = rows ? (int64_t)tm * C::UMMA_M + cta_rank * BM_CTA + i * 32 + lane
                                     : (int64_t)tn * C::UMMA_N + (COLVEC ? i * 32 + lane : lane * C::ACC);
                    const ScaleView& v = rows ? p.sa : p.sb;
                    const bool ok = i < (rows ? NA : NB) && r < (rows ? p.M : p.N) && (rows || COLVEC || lane < 2);
                    if (ok) exists |= 1u << i; else r = 0;
                    src[i] = v.p + (r >> v.shift) * v.rs;
                }
                const int64_t ks = rows ? p.sa.ks : p.sb.ks;
                for (int kb = 0; kb < p.num_kb; ++kb) {
                    if (!warp_wait(sempty_bar(slot), phase ^ 1u, p, 1500 + slot, t)) { alive = false; break; }
                    const uint32_t dst = ring + (uint32_t)(slot * C::SLOT_FLOATS + (rows ? 0 : BM_CTA) + lane) * 4u;
#pragma unroll
                    for (int i = 0; i < NMOST; ++i) {
                        if (i < (rows ? NA : NB)) cp_async4(dst + i * 128u, src[i], (exists >> i) & 1u);
                        src[i] += ks;
                    }
                    cp_async_arrive(sfull_bar(slot));
                    if (++slot == SLOTS) { slot = 0; phase ^= 1u; }
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        }
    } else {
        /* ------------------------------------------------------------ epilogue -------- */
        if constexpr (C::REALLOC) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        const int q = warp & 3, eh = (warp - 4) >> 2;
        const uint32_t tlane = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(eh * C::ACC);
        int unit = 0, slot = 0; uint32_t sphase = 0;
        bool alive = true;
        for (int t = cluster_id; t < num_tiles && alive; t += num_clusters) {
            int tm, tn; tile_coords(t, p.tiles_m, p.tiles_n, p.tile_group, tm, tn);
            uint64_t sum[C::ACC / 2];
#pragma unroll
            for (int c = 0; c < C::ACC / 2; ++c) sum[c] = 0;
            for (int kb = 0; kb < p.num_kb; ++kb, ++unit) {
                const int acc = unit & 1;
                if (!warp_wait(sfull_bar(slot), sphase, p, 1600 + slot, t)) { alive = false; break; }
                const uint32_t sc = ring + (uint32_t)(slot * C::SLOT_FLOATS) * 4u;
                float sr, sh = 1.0f;
                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(sr) : "r"(sc + (uint32_t)(q * 32 + lane) * 4u) : "memory");
                if (!COLVEC) {
                    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(sh) : "r"(sc + (uint32_t)(BM_CTA + eh) * 4u) : "memory");
                    sr *= sh;
                }
                const uint64_t s2 = pack2(sr, sr);
                if (!warp_wait(tfull_bar(acc), (uint32_t)(unit >> 1) & 1u, p, 1400 + acc, t)) { alive = false; break; }
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < C::ACC; c += 32) {
                    float v[32];
                    tmem_ld_32x32(tlane + (uint32_t)(acc * C::UMMA_N + c), v);
                    tmem_ld_wait();
                    if (COLVEC) {
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            uint64_t c01, c23;
                            asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(c01), "=l"(c23)
                                         : "r"(sc + (uint32_t)(BM_CTA + eh * C::ACC + c + j) * 4u) : "memory");
                            sum[(c + j) / 2] = fma2(pack2(v[j], v[j + 1]), mul2(c01, s2), sum[(c + j) / 2]);
                            sum[(c + j) / 2 + 1] = fma2(pack2(v[j + 2], v[j + 3]), mul2(c23, s2), sum[(c + j) / 2 + 1]);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; j += 2) sum[(c + j) / 2] = fma2(pack2(v[j], v[j + 1]), s2, sum[(c + j) / 2]);
                    }
                }
                /* block taken: hand the buffer (in the leader CTA) and the scales' slot back */
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (CTAS == 1) mbar_arrive_cluster(tempty_bar(acc));
                    else           mbar_arrive_cluster(mapa(tempty_bar(acc), 0));
                    mbar_arrive(sempty_bar(slot));
                }
                if (++slot == SLOTS) { slot = 0; sphase ^= 1u; }
            }
            if (!alive) break;
            const int64_t row = (int64_t)tm * C::UMMA_M + cta_rank * BM_CTA + q * 32 + lane;
            const int64_t col0 = (int64_t)tn * C::UMMA_N + eh * C::ACC;
            if (row < p.M) {
#pragma unroll
                for (int c = 0; c < C::ACC; c += 8) {
                    float v[8];
#pragma unroll
                    for (int j = 0; j < 8; j += 2) unpack2(sum[(c + j) / 2], v[j], v[j + 1]);
                    if (p.d_type == DECXB_F32)      store_row8<float>(p, row, col0 + c, v);
                    else if (p.d_type == DECXB_F16) store_row8<__half>(p, row, col0 + c, v);
                    else                            store_row8<__nv_bfloat16>(p, row, col0 + c, v);
                }
            }
        }
    }

    /* ---------------------------------------------------------------- teardown -------- */
    tc_fence_before();
    __syncthreads();
    if (CTAS == 2) cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc<CTAS>(tmem_base, C::TMEM_COLS);
    }
}

/* ------------------------------------------------------------------ host side -------- */
/* rows x K codes with K contiguous and a row pitch of `ld` bytes; box = 128 codes x box_rows. */
int make_map_fp8(decxb_ctx* ctx, CUtensorMap* map, const void* base, int64_t rows, int64_t K, int64_t ld, int box_rows)
{
    auto fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(decxb_tensor_map_encoder());
    if (!fn) return decxb_fail(ctx, DECXB_ERR_CUDA, "cuTensorMapEncodeTiled entry point not found");
    cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld};
    cuuint32_t box[2] = {(cuuint32_t)BK, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return decxb_fail(ctx, DECXB_ERR_CUDA, "cuTensorMapEncodeTiled (fp8) failed: " + std::to_string((int)r));
    return DECXB_OK;
}

template <int CTAS, int BN, bool COLVEC>
int launch(decxb_ctx* ctx, const decxb_fp8_matrix& A, const decxb_fp8_matrix& B, Params p, cudaStream_t s)
{
    using C = Cfg<CTAS, BN, COLVEC>;
    auto kernel = decxb_gemm_fp8_kernel<CTAS, BN, COLVEC>;
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
    if (C::REALLOC && regs[dev] != 168) return decxb_fail(ctx, DECXB_ERR_CUDA, "fp8 GEMM kernel was not compiled to 168 registers");
    CUtensorMap ma, mb;
    int rc;
    if ((rc = make_map_fp8(ctx, &ma, A.data, A.rows, A.cols, A.ld, BM_CTA))) return rc;
    if ((rc = make_map_fp8(ctx, &mb, B.data, B.rows, B.cols, B.ld, BN))) return rc;
    const int64_t tm = decxb_ceil_div(p.M, C::UMMA_M), tn = decxb_ceil_div(p.N, C::UMMA_N);
    if (tm * tn > 0x7fffffffLL) return decxb_fail(ctx, DECXB_ERR_TOO_LARGE, "fp8 gemm tiles");
    p.tiles_m = (int)tm; p.tiles_n = (int)tn;
    p.idesc = make_idesc_fp8(C::UMMA_M, C::UMMA_N, A.type, B.type);
    int64_t clusters = (ctx->sm_count - ctx->reserved_sms) / CTAS;
    if (clusters > tm * tn) clusters = tm * tn;
    if (clusters < 1) clusters = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(clusters * CTAS), 1, 1);
    cfg.blockDim = dim3(THREADS, 1, 1);
    cfg.dynamicSmemBytes = C::SMEM_BYTES;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CTAS; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = 1;
    decxb_launch_scope scope(ctx, s, DECXB_K_GEMM);
    DECXB_CUDA_TRY(ctx, cudaLaunchKernelEx(&cfg, kernel, ma, mb, p));
    return DECXB_OK;
}

/* Codes that the copy engine cannot address are copied to a pitch it can. */
int reachable(decxb_ctx* ctx, decxb_fp8_matrix* m, void** scratch, cudaStream_t s)
{
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
        p.tile_group = 8;
        p.sa = view_of(A); p.sb = view_of(B);
        p.C = C; p.ldc = ldc; p.D = D; p.ldd = ldd; p.d_type = d_type;
        p.d_vec = aligned(D, ldd * e, 16);
        p.c_vec = C && aligned(C, ldc * e, 16);
        p.wait_limit_ns = ctx->wait_limit_ns; p.status = ctx->d_status;
        rc = B.block_rows == 1 ? launch<1, 128, true>(ctx, A, B, p, s) : launch<1, 128, false>(ctx, A, B, p, s);
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
} catch (const std::bad_alloc&) { return DECXB_ERR_ALLOC; }
