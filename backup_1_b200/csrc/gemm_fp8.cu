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
    bool tma_store;                /* D leaves through the copy engine                 */
    long long wait_limit_ns;
    decxb_dev_status* status;
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
            bool give_up = false;
            if (elect_one()) {
                const unsigned long long t = globaltimer_ns();
                if (t0 == 0) t0 = t;
                give_up = *reinterpret_cast<volatile int*>(&p.status->code) != 0;
                if (!give_up && (long long)(t - t0) > p.wait_limit_ns) {
                    give_up = true;
                    if (atomicCAS(&p.status->code, 0, DECXB_DEVERR_WAIT_EXPIRED) == 0) {
                        p.status->where = where; p.status->block = (int)blockIdx.x; p.status->detail = detail;
                        __threadfence_system();
                    }
                }
            }
            if (__any_sync(0xffffffffu, give_up)) return false;
        }
    }
    return true;
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
/* Arrival on the leader CTA's barrier.  What it releases are reads of tensor memory, which tcgen05.wait::ld and the
 * tcgen05 fence before it have ordered; a release at cluster scope would add a memory fence of about a thousand
 * clocks, twice a k-block's arithmetic. */
__device__ __forceinline__ void mbar_arrive_leader(uint32_t bar)
{
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" :: "r"(mapa(bar, 0)) : "memory");
}

__device__ __forceinline__ float lds_f32(uint32_t at)
{
    float v; asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory"); return v;
}

__device__ __forceinline__ float4 lds_f32x4(uint32_t at)
{
    float4 v; asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory"); return v;
}

/* tcgen05.wait::ld with the loaded registers as operands: nothing that reads them can be moved ahead of it. */
__device__ __forceinline__ void tmem_ld_wait32(float* v)
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]),
                   "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]) :: "memory");
    asm volatile("" : "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]),
                      "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31]) :: "memory");
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
 * Through the copy engine: `n` 16-byte pieces of this row (8 of them fill the box), then one store of the box. */
template <typename T>
__device__ __forceinline__ void box_pieces(uint32_t box, int lane, int first, const float* v)
{
    constexpr int E = 16 / sizeof(T);
#pragma unroll
    for (int j = 0; j < 32; j += E) {
        uint4 u;
        T* e = reinterpret_cast<T*>(&u);
#pragma unroll
        for (int k = 0; k < E; ++k) e[k] = from_f32<T>(v[j + k]);
        const uint32_t at = box + (uint32_t)lane * 128u + (uint32_t)(((first + j / E) ^ (lane & 7)) << 4);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" :: "r"(at), "r"(u.x), "r"(u.y), "r"(u.z), "r"(u.w) : "memory");
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
    static constexpr int KB_FLOATS = BM_CTA + (COLVEC ? UMMA_N : 32);
    static constexpr int SCALE_BYTES = SLOTS * KB_FLOATS * 4;
    static constexpr int BOX_BYTES = EPI_WARPS * 4096;         /* result boxes, one a warp */
    static constexpr int STAGES_RAW = (SMEM_LIMIT - 2048 - SCALE_BYTES - BOX_BYTES) / STAGE_BYTES;
    static constexpr int STAGES = STAGES_RAW > 8 ? 8 : STAGES_RAW;
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + BOX_BYTES + SCALE_BYTES + 1024 /* alignment slack */ + 512 /* barriers */;
    static constexpr int BUFS = 512 / UMMA_N > 4 ? 4 : 512 / UMMA_N;      /* accumulators in tensor memory */
    static constexpr int TMEM_COLS = BUFS * UMMA_N;
    /* 128 running sums per thread need the registers of warp group 0: see the launch */
    static constexpr bool REALLOC = ACC > 64;
    static_assert(UMMA_N % 64 == 0 && UMMA_N <= 256 && ACC <= 128, "tile width");
    static_assert(SMEM_BYTES <= SMEM_LIMIT, "shared memory");
    static_assert(BUFS == 2 || BUFS == 4, "buffers alternate between two issuers");
    /* the epilogue reads a stage's barrier by parity and lies at most BUFS k-blocks behind the issuers */
    static_assert(STAGES > BUFS, "a stage's barrier must not turn over twice unseen");
};

template <int CTAS, int BN, bool COLVEC>
__global__ void __launch_bounds__(THREADS, 1)
decxb_gemm_fp8_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                      const __grid_constant__ CUtensorMap map_d, const Params p)
{
    using C = Cfg<CTAS, BN, COLVEC>;
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
    const uint32_t tmem_slot = bars + 8u * (2 * C::STAGES + C::BUFS + 2 * SLOTS);
    auto stage_a = [&](int s) { return smem_base + s * C::STAGE_BYTES; };
    auto stage_b = [&](int s) { return smem_base + s * C::STAGE_BYTES + C::A_BYTES; };

    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t cta_rank = CTAS == 2 ? cluster_ctarank() : 0u;
    const bool is_leader = cta_rank == 0;
    const int cluster_id = (int)blockIdx.x / CTAS, num_clusters = (int)gridDim.x / CTAS;
    const int num_tiles = p.tiles_m * p.tiles_n;

    if (threadIdx.x == 0) {
        prefetch_tensormap(&map_a); prefetch_tensormap(&map_b);
        if (p.tma_store) prefetch_tensormap(&map_d);
        for (int s = 0; s < C::STAGES; ++s) { mbar_init(full_bar(s), 1); mbar_init(done_bar(s), 1); }
        for (int b = 0; b < C::BUFS; ++b) mbar_init(tempty_bar(b), EPI_WARPS * CTAS);
        for (int s = 0; s < SLOTS; ++s) { mbar_init(sfull_bar(s), 32); mbar_init(sempty_bar(s), EPI_WARPS); }
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
            int stage = 0; uint32_t phase = 0;
            uint32_t armed = 0, armed_parity = 0;
            bool alive = true;
            for (int t = cluster_id; t < num_tiles && alive; t += num_clusters) {
                int tm, tn; tile_coords(t, p.tiles_m, p.tiles_n, p.tile_group, tm, tn);
                const int row_a = tm * C::UMMA_M + (int)cta_rank * BM_CTA;
                const int row_b = tn * C::UMMA_N + (int)cta_rank * BN;
                for (int kb = 0; kb < p.num_kb; ++kb) {
                    if (!warp_wait(done_bar(stage), phase ^ 1u, p, 1100 + stage, t)) { alive = false; break; }
                    if (elect_one()) {
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
                    }
                    __syncwarp();
                    armed |= 1u << stage;
                    armed_parity = (armed_parity & ~(1u << stage)) | (phase << stage);
                    if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
                }
            }
            /* a wait gave up somewhere: wait (with a limit) for the copies that are still on their way into
             * shared memory; the leader's barriers count its peer's as well */
            if (is_leader && lane == 0 && *reinterpret_cast<volatile int*>(&p.status->code) != 0) {
                for (int s2 = 0; s2 < C::STAGES; ++s2) {
                    if (!((armed >> s2) & 1u)) continue;
                    for (int tries = 0; tries < 2048 && !mbar_try_wait(full_bar(s2), (armed_parity >> s2) & 1u); ++tries)
                        __nanosleep(64);
                }
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
                        if (elect_one()) {
                            const uint32_t tmem_d = tmem_base + (uint32_t)(acc * C::UMMA_N);
                            const uint64_t da = make_smem_desc(stage_a(stage)), db = make_smem_desc(stage_b(stage));
#pragma unroll
                            for (int kk = 0; kk < BK / UMMA_K; ++kk) {
                                const uint64_t koff = (uint64_t)((kk * UMMA_K) >> 4);
                                umma_fp8<CTAS>(tmem_d, da + koff, db + koff, p.idesc, kk != 0 ? 1u : 0u);
                            }
                            umma_commit<CTAS>(done_bar(stage));
                        }
                        __syncwarp();
                        if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
                    }
                }
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
        if constexpr (C::REALLOC) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        const int q = warp & 3, eh = (warp - 4) >> 2;
        const uint32_t tlane = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(eh * C::ACC);
        const uint32_t box = boxes + (uint32_t)(warp - 4) * 4096u;
        int unit = 0, slot = 0, stage = 0;
        uint32_t sphase = 0, phase = 0;
        bool alive = true;
        for (int t = cluster_id; t < num_tiles && alive; t += num_clusters) {
            int tm, tn; tile_coords(t, p.tiles_m, p.tiles_n, p.tile_group, tm, tn);
            float sum[C::ACC];
#pragma unroll
            for (int c = 0; c < C::ACC; ++c) sum[c] = 0.0f;
            for (int kb = 0; kb < p.num_kb; ++kb, ++unit) {
                const int acc = unit % C::BUFS;
                if (!warp_wait(sfull_bar(slot), sphase, p, 1600 + slot, t)) { alive = false; break; }
                const uint32_t sc = ring + (uint32_t)(slot * C::KB_FLOATS) * 4u;
                float sr = lds_f32(sc + (uint32_t)(q * 32 + lane) * 4u);
                if (!COLVEC) sr *= lds_f32(sc + (uint32_t)(BM_CTA + eh) * 4u);
                if (!warp_wait(done_bar(stage), phase, p, 1400 + stage, t)) { alive = false; break; }
                tc_fence_after();
                /* 32 columns are multiplied while the next 32 are on their way */
                float v[2][32];
                tmem_ld_32x32(tlane + (uint32_t)(acc * C::UMMA_N), v[0]);
#pragma unroll
                for (int c = 0; c < C::ACC; c += 32) {
                    float* w = v[(c >> 5) & 1];
                    tmem_ld_wait32(w);
                    if (c + 32 < C::ACC) tmem_ld_32x32(tlane + (uint32_t)(acc * C::UMMA_N + c + 32), v[((c >> 5) + 1) & 1]);
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        float4 f = make_float4(sr, sr, sr, sr);
                        if (COLVEC) {
                            const float4 g = lds_f32x4(sc + (uint32_t)(BM_CTA + eh * C::ACC + c + j) * 4u);
                            f.x *= g.x; f.y *= g.y; f.z *= g.z; f.w *= g.w;
                        }
                        sum[c + j] = fmaf(w[j], f.x, sum[c + j]);
                        sum[c + j + 1] = fmaf(w[j + 1], f.y, sum[c + j + 1]);
                        sum[c + j + 2] = fmaf(w[j + 2], f.z, sum[c + j + 2]);
                        sum[c + j + 3] = fmaf(w[j + 3], f.w, sum[c + j + 3]);
                    }
                }
                /* block taken: hand the buffer (in the leader CTA) and the scales' slot back */
                tc_fence_before();
                __syncwarp();
                if (elect_one()) {
                    if (CTAS == 1 || is_leader) mbar_arrive(tempty_bar(acc));
                    else                        mbar_arrive_leader(tempty_bar(acc));
                    mbar_arrive(sempty_bar(slot));
                }
                __syncwarp();
                if (++slot == SLOTS) { slot = 0; sphase ^= 1u; }
                if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
            }
            if (!alive) break;
            const int64_t row0 = (int64_t)tm * C::UMMA_M + cta_rank * BM_CTA + q * 32;
            const int64_t col0 = (int64_t)tn * C::UMMA_N + eh * C::ACC;
            if (row0 >= p.M) continue;
#pragma unroll
            for (int c = 0; c < C::ACC; c += 32) {
                if (col0 + c >= p.N) break;
                const float* v = sum + c;
                const bool narrow = p.d_type != DECXB_F32;        /* 64 columns fill a box */
                if (p.tma_store) {
                    const int first = narrow && (c & 32) ? 4 : 0;
                    if (first == 0) {
                        if (lane == 0) tma_store_wait_read<0>();      /* the box before has been read */
                        __syncwarp();
                    }
                    if (!narrow)                        box_pieces<float>(box, lane, 0, v);
                    else if (p.d_type == DECXB_F16)     box_pieces<__half>(box, lane, first, v);
                    else                                box_pieces<__nv_bfloat16>(box, lane, first, v);
                    if (!narrow || first || col0 + c + 32 >= p.N) {
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            tma_store_2d(&map_d, box, (int)(col0 + (narrow ? (c & ~63) : c)), (int)row0);
                            tma_store_commit();
                        }
                    }
                } else {
                    __syncwarp();
                    box_pieces<float>(box, lane, 0, v);
                    __syncwarp();
                    if (!narrow)                        box_rows<float>(p, box, lane, row0, col0 + c + lane);
                    else if (p.d_type == DECXB_F16)     box_rows<__half>(p, box, lane, row0, col0 + c + lane);
                    else                                box_rows<__nv_bfloat16>(p, box, lane, row0, col0 + c + lane);
                }
            }
        }
        if (p.tma_store && lane == 0) tma_store_wait_all();       /* the box stays until the copy engine is done */
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
    if ((rc = make_map_fp8(ctx, &ma, A, BM_CTA)) || (rc = make_map_fp8(ctx, &mb, B, BN))) return rc;
    CUtensorMap md = ma;
    if (p.tma_store) {
        const int e = size_of(p.d_type);
        const CUtensorMapDataType type = p.d_type == DECXB_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                       : p.d_type == DECXB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
        if ((rc = make_map_2d(ctx, &md, type, e, p.D, p.M, p.N, p.ldd, 32))) return rc;
    }
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
    DECXB_CUDA_TRY(ctx, cudaLaunchKernelEx(&cfg, kernel, ma, mb, md, p));
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
        /* the copy engine clips a store at the array's edge in whole 16-byte pieces, so N has to be made of them too */
        p.tma_store = !C && aligned(D, ldd * e, 16) && N * e % 16 == 0;
        p.wait_limit_ns = ctx->wait_limit_ns; p.status = ctx->d_status;
        const bool by_row = B.block_rows == 1;
        const int64_t pairs = decxb_ceil_div(M, 256) * decxb_ceil_div(N, 256);
        if (pairs * 2 >= ctx->sm_count / 2)
            rc = by_row ? launch<2, 128, true>(ctx, A, B, p, s) : launch<2, 128, false>(ctx, A, B, p, s);
        else
            rc = by_row ? launch<1, 128, true>(ctx, A, B, p, s) : launch<1, 128, false>(ctx, A, B, p, s);
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
