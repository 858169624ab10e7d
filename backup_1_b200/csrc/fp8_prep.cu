/*
 * What feeds the 8-bit product (sm_100a): quantisation of a matrix as it stands and transposed, the
 * root-mean-square norm with the residual's addition and an fp8 output, and the norm's backward pass.
 * All of them are bound by memory: every array is read once and written once.
 */
#include "fp8.cuh"
#include "tc_ptx.cuh"

#include <mutex>

namespace {

using namespace fp8;

__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

/* Every kernel here may start while the one before it in the stream drains, and waits for its memory here. */
__device__ __forceinline__ void start_after_previous()
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

template <typename... P, typename... A>
int launch_after(decxb_ctx* ctx, void (*kernel)(P...), unsigned grid, dim3 threads, size_t smem, cudaStream_t s, const A&... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, 1, 1); cfg.blockDim = threads; cfg.dynamicSmemBytes = smem; cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 1;
    decxb_launch_scope scope(ctx, s, DECXB_K_SPLIT);
    DECXB_CUDA_TRY(ctx, cudaLaunchKernelEx(&cfg, kernel, args...));
    return DECXB_OK;
}

/* Bulk copy of `bytes` (a multiple of 16, both addresses too) to shared memory, counted on an mbarrier. */
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 :: "r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

/* Wait for a stage's copies.  False where they did not come within the limit, or another wait of the launch had given up before. */
__device__ __forceinline__ bool wait_copy(uint32_t bar, uint32_t parity, const Waits& w)
{
    unsigned long long t0 = 0;
    for (uint32_t spins = 1; !tcptx::mbar_try_wait(bar, parity); ++spins) {
        if (spins & 1023u) continue;
        if (gave_up(w)) return false;
        const unsigned long long t = tcptx::globaltimer_ns();
        if (t0 == 0) t0 = t;
        if ((long long)(t - t0) > w.limit_ns) {
            give_up(w, 3000, 0);
            return false;
        }
    }
    return true;
}

/* By the thread that fetches, when a block leaves its rows early: waits (with a limit) for the copies of `row` and of the
 * stages behind it, which may still be on their way into the block's shared memory. */
__device__ __forceinline__ void drain_copies(uint64_t* bars, int stages, int st, uint32_t phase, int64_t row, int64_t rows)
{
    for (int i = 0; i < stages && row < rows; ++i, row += gridDim.x) {
        for (int tries = 0; tries < 2048 && !tcptx::mbar_try_wait(tcptx::smem_u32(&bars[st]), phase); ++tries) __nanosleep(64);
        if (++st == stages) { st = 0; phase ^= 1u; }
    }
}

/* ---- root-mean-square norm ---------------------------------------------------------------
 * One block per row, or eight rows of up to 256 columns with a warp each.  A thread holds VPT vectors of eight consecutive
 * columns, vector i * blockDim + tid, so the 16 lanes of half a warp cover one 128-column block of the row and its
 * largest magnitude is four shuffles away. */
struct NormArgs {
    int64_t rows, cols;
    const void *x, *r, *gamma; void *h, *y;
    int64_t ldx, ldr, ldh, ldy;
    int gamma_type, rule;
    float eps;
    bool vec, gvec;                   /* 128-bit accesses to x, r, h, y / gamma                     */
    uint8_t* q; int64_t ldq; float* s; int64_t srs, sbs; int qtype; bool qvec;
};

/* Quantises the `n` columns (eight, but at a ragged row's end) from `c` on of one row: the 16 lanes of the block agree on its scale. */
__device__ __forceinline__ void quantise_row8(const NormArgs& a, uint8_t* q, float* scales, int c, int n, const float* y)
{
    float amax = fabsf(y[0]);                  /* columns that do not exist are zeros */
#pragma unroll
    for (int j = 1; j < 8; ++j) amax = max_nan(amax, fabsf(y[j]));
#pragma unroll
    for (int o = 8; o; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (n <= 0) return;
    const float s = scale_of(amax, a.qtype, a.rule);
    const Quantiser z = quantiser(s);
    store_codes8(q + c, n, a.qvec, a.qtype == DECXB_FP8_E4M3 ? codes8<DECXB_FP8_E4M3>(y, z) : codes8<DECXB_FP8_E5M2>(y, z));
    if ((c & 127) == 0) scales[(c >> 7) * a.sbs] = s;
}

/* WHOLE: every vector of the row lies in it and every array takes 128-bit accesses (the checks cost a third of the kernel's
 * instructions, which bound it for 16-bit types). */
template <typename T, int VPT, bool WHOLE>
__global__ void __launch_bounds__(1024, VPT <= 2 ? 2 : 1)
decxb_rmsnorm_kernel(const NormArgs a)
{
    __shared__ float part[32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, nwarps = blockDim.x >> 5;
    const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    const int cols = (int)a.cols;
    if (row >= a.rows) return;             /* a whole warp, in a block without barriers */
    const bool vec = WHOLE || a.vec, gvec = WHOLE || a.gvec;
    auto count = [&](int c) { return WHOLE ? (c < cols ? 8 : 0) : min(8, cols - c); };
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    float v[VPT][8];
    float sum = 0.0f;
    start_after_previous();
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int c = (i * (int)blockDim.x + tid) * 8;
        load8(x + c, count(c), vec, v[i]);
    }
    if (a.r) {
        const T* r = static_cast<const T*>(a.r) + row * a.ldr;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = (i * (int)blockDim.x + tid) * 8;
            float w[8];
            load8(r + c, count(c), vec, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] += w[j];
        }
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = fmaf(v[i][j], v[i][j], sum);
    sum = warp_sum(sum);
    if (nwarps > 1) {
        if (lane == 0) part[warp] = sum;
        __syncthreads();
        sum = warp_sum(lane < nwarps ? part[lane] : 0.0f);
    }
    const float rstd = rsqrtf(sum / (float)cols + a.eps);
    if (a.h) {
        T* h = static_cast<T*>(a.h) + row * a.ldh;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = (i * (int)blockDim.x + tid) * 8;
            if (count(c) > 0) store8(h + c, count(c), vec, v[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int c = (i * (int)blockDim.x + tid) * 8;
        float g[8];
        load8_any(a.gamma, a.gamma_type, c, count(c), gvec, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] * rstd * g[j];
        if (a.y && count(c) > 0) store8(static_cast<T*>(a.y) + row * a.ldy + c, count(c), vec, v[i]);
        if (a.q) quantise_row8(a, a.q + row * a.ldq, a.s + row * a.srs, c, count(c), v[i]);
    }
}

/* Many rows of up to 4096 columns: a block walks rows blockIdx, blockIdx + gridDim, ... that bulk copies bring to shared memory
 * `stages` rows ahead, one vector a thread.  Against a block per row (above) there is always something on the way, and
 * what does not depend on the row (gamma, addresses) is done once: the instructions of 16-bit rows bound that
 * kernel (43 an element, 73 % of the issue slots).
 * Two blocks to an SM, each two rows ahead: 52.1 us for 8192 x 4096 with the sum, the plain and the fp8 output (5.8 TB/s in a graph; called
 * one after another 54 to 56, singly on an idle device 63). Before the blocks asked whether a row had come it was 51.1, and then
 * four rows ahead 52.5, three blocks 56, and compiled for the registers of two blocks 64, with the same counts of
 * instructions: reads and writes share the memory best when neither runs far ahead. */
template <typename T>
__global__ void __launch_bounds__(512, 3)
decxb_rmsnorm_rows_kernel(const NormArgs a, const int stages, const Waits waits)
{
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float part[2][17];              /* [16]: not 0 where a thread gave its wait up */
    __shared__ __align__(8) uint64_t bars[8];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, nwarps = blockDim.x >> 5, cols = (int)a.cols;
    const int arrays = a.r ? 2 : 1;
    const uint32_t row_bytes = (uint32_t)cols * (uint32_t)sizeof(T);
    const int first = tid * 8, n = first < cols ? 8 : 0;
    auto fetch = [&](int64_t row, int st) {
        const uint32_t bar = tcptx::smem_u32(&bars[st]), at = tcptx::smem_u32(smem) + (uint32_t)(st * arrays) * row_bytes;
        tcptx::mbar_arrive_expect_tx(bar, row_bytes * arrays);
        if (row == waits.lost) return;
        bulk_load(at, static_cast<const T*>(a.x) + row * a.ldx, row_bytes, bar);
        if (a.r) bulk_load(at + row_bytes, static_cast<const T*>(a.r) + row * a.ldr, row_bytes, bar);
    };
    if (tid == 0) {
        part[0][16] = part[1][16] = 0.0f;
        for (int st = 0; st < stages; ++st) tcptx::mbar_init(tcptx::smem_u32(&bars[st]), 1);
        tcptx::fence_barrier_init();
    }
    __syncthreads();
    start_after_previous();
    if (tid == 0)
        for (int st = 0; st < stages; ++st)
            if (blockIdx.x + (int64_t)st * gridDim.x < a.rows) fetch(blockIdx.x + (int64_t)st * gridDim.x, st);
    float g[8];
    load8_any(a.gamma, a.gamma_type, first, n, true, g);
    const float of_cols = 1.0f / (float)cols;
    int st = 0, turn = 0; uint32_t phase = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
        if (!wait_copy(tcptx::smem_u32(&bars[st]), phase, waits)) part[turn][16] = 1.0f;
        const T* in = reinterpret_cast<const T*>(smem + (size_t)(st * arrays) * row_bytes);
        float v[8], sum = 0.0f;
        load8(in + first, n, true, v);
        if (a.r) {
            float w[8];
            load8(in + cols + first, n, true, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += w[j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = fmaf(v[j], v[j], sum);
        sum = warp_sum(sum);
        if (lane == 0) part[turn][warp] = sum;
        __syncthreads();                       /* every thread has its values: the stage can be filled again */
        if (part[turn][16] != 0.0f) {          /* the row did not come: it and those behind it stay unwritten */
            if (tid == 0) drain_copies(bars, stages, st, phase, row, a.rows);
            return;
        }
        if (tid == 0 && row + (int64_t)stages * gridDim.x < a.rows) fetch(row + (int64_t)stages * gridDim.x, st);
        const float rstd = rsqrtf(warp_sum(lane < nwarps ? part[turn][lane] : 0.0f) * of_cols + a.eps);
        if (a.h && n) store8(static_cast<T*>(a.h) + row * a.ldh + first, 8, true, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = v[j] * rstd * g[j];
        if (a.y && n) store8(static_cast<T*>(a.y) + row * a.ldy + first, 8, true, v);
        if (a.q) quantise_row8(a, a.q + row * a.ldq, a.s + row * a.srs, first, n, v);
        if (++st == stages) { st = 0; phase ^= 1u; }
    }
}

/* Rows too long for the registers: the row is read twice (the second time from L2, mostly). */
template <typename T>
__global__ void __launch_bounds__(1024)
decxb_rmsnorm_wide_kernel(const NormArgs a)
{
    __shared__ float part[32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, nwarps = blockDim.x >> 5;
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* r = a.r ? static_cast<const T*>(a.r) + row * a.ldr : nullptr;
    start_after_previous();
    float sum = 0.0f, v[8], w[8];
    for (int64_t c = (int64_t)tid * 8; c < a.cols; c += (int64_t)blockDim.x * 8) {
        const int n = (int)min((int64_t)8, a.cols - c);
        load8(x + c, n, a.vec, v);
        if (r) {
            load8(r + c, n, a.vec, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += w[j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = fmaf(v[j], v[j], sum);
    }
    sum = warp_sum(sum);
    if (lane == 0) part[warp] = sum;
    __syncthreads();
    sum = warp_sum(lane < nwarps ? part[lane] : 0.0f);
    const float rstd = rsqrtf(sum / (float)a.cols + a.eps);
    /* whole warps go round together (the quantisation exchanges values inside a warp) */
    for (int64_t c0 = (int64_t)warp * 256; c0 < a.cols; c0 += (int64_t)blockDim.x * 8) {
        const int64_t c = c0 + lane * 8;
        const int n = (int)min((int64_t)8, a.cols - c);
        load8(x + c, n, a.vec, v);
        if (r) {
            load8(r + c, n, a.vec, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += w[j];
        }
        if (a.h && n > 0) store8(static_cast<T*>(a.h) + row * a.ldh + c, n, a.vec, v);
        load8_any(a.gamma, a.gamma_type, c, n, a.gvec, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = v[j] * rstd * w[j];
        if (a.y && n > 0) store8(static_cast<T*>(a.y) + row * a.ldy + c, n, a.vec, v);
        if (a.q) quantise_row8(a, a.q + row * a.ldq, a.s + row * a.srs, (int)c, n, v);
    }
}

/* Threads per row: multiples of 32 that cover `nvec` vectors with at most `vpt` each. */
int threads_for(int64_t nvec, int vpt, int most)
{
    int64_t t = decxb_ceil_to(decxb_ceil_div(nvec, vpt), 32);
    return (int)(t > most ? most : t < 32 ? 32 : t);
}

template <typename T, int VPT>
int launch_norm_rows(decxb_ctx* ctx, const NormArgs& a, int64_t nvec, cudaStream_t s)
{
    const bool whole = a.vec && a.gvec && a.cols % 8 == 0 && (!a.q || a.qvec);
    const unsigned threads = (unsigned)threads_for(nvec, VPT, 1024), rows = threads == 32 ? 8 : 1;
    const unsigned grid = (unsigned)decxb_ceil_div(a.rows, rows);
    return whole ? launch_after(ctx, decxb_rmsnorm_kernel<T, VPT, true>, grid, dim3(threads, rows), 0, s, a)
                 : launch_after(ctx, decxb_rmsnorm_kernel<T, VPT, false>, grid, dim3(threads, rows), 0, s, a);
}

template <typename T>
int launch_norm_many(decxb_ctx* ctx, const NormArgs& a, cudaStream_t s)
{
    auto kernel = decxb_rmsnorm_rows_kernel<T>;
    const int stages = 2;
    const size_t smem = (size_t)stages * a.cols * sizeof(T) * (a.r ? 2 : 1);      /* at most 32 KiB */
    static std::once_flag once[DECXB_MAX_DEVICES];
    static cudaError_t err[DECXB_MAX_DEVICES];
    std::call_once(once[ctx->device], [&] { err[ctx->device] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 32 * 1024); });
    if (err[ctx->device] != cudaSuccess) return decxb_fail(ctx, DECXB_ERR_CUDA, std::string("norm kernel attributes: ") + cudaGetErrorString(err[ctx->device]));
    return launch_after(ctx, kernel, (unsigned)(2 * ctx->sm_count), threads_for(decxb_ceil_div(a.cols, 8), 1, 512), smem, s, a, stages,
                        waits_of(ctx));
}

/* One vector a thread as far as 1024 threads reach (8192 x 4096 bf16 with one, two, four: 64, 69, 74 us): a block's loads,
 * sum and stores follow one another, so it is the number of blocks on an SM that keeps the memory busy. */
template <typename T>
int launch_norm(decxb_ctx* ctx, const NormArgs& a, cudaStream_t s)
{
    const int64_t nvec = decxb_ceil_div(a.cols, 8);
    /* 16-bit rows of 2049 to 4096 columns, eight or more to an SM: 8192 x 4096 60.6 us with a block a row, 52.1 with rows by bulk
     * copies; but 600 x 4096 5.6 and 7.0, 16384 x 1024 29 and 58, 4096 x 4096 fp32 46.6 and 53.8 */
    if constexpr (sizeof(T) == 2)
        if (a.vec && a.gvec && a.cols % 8 == 0 && (!a.q || a.qvec) && a.cols > 2048 && a.cols <= 4096 && a.rows >= 8 * (int64_t)ctx->sm_count)
            return launch_norm_many<T>(ctx, a, s);
    if (nvec <= 1024) return launch_norm_rows<T, 1>(ctx, a, nvec, s);
    if (nvec <= 2048) return launch_norm_rows<T, 2>(ctx, a, nvec, s);
    if (nvec <= 4096) return launch_norm_rows<T, 4>(ctx, a, nvec, s);
    return launch_after(ctx, decxb_rmsnorm_wide_kernel<T>, (unsigned)a.rows, 1024, 0, s, a);
}

/* ---- its backward pass ---------------------------------------------------------------------
 * A thread keeps the same columns throughout and sums their share of dgamma in registers.  Each block leaves its sums in
 * its own row of the workspace, and a second kernel adds the rows in ascending order: no atomics, the same bits every
 * time.  Rows up to 256 columns belong to a warp, longer ones to a block. */
struct NormBwdArgs {
    int64_t rows, cols;
    const void *dy, *h, *dr, *gamma; void* dx;
    int64_t lddy, ldh, lddr, lddx;
    int gamma_type;
    float eps;
    bool vec, gvec;
    float* part;                      /* [gridDim][cols], or NULL                                    */
};

/* Sums of (a, b) over the block; `buf` alternates between rows so that one barrier a row is enough. */
__device__ __forceinline__ float2 block_sum2(float a, float b, float2* buf, int warp, int lane, int nwarps)
{
    a = warp_sum(a); b = warp_sum(b);
    if (lane == 0) buf[warp] = make_float2(a, b);
    __syncthreads();
    const float2 p = lane < nwarps ? buf[lane] : make_float2(0.0f, 0.0f);
    return make_float2(warp_sum(p.x), warp_sum(p.y));
}

/* dX of eight columns, and their share of dgamma on top of `acc`: w = dY, o = dR on entry and dX on return. */
__device__ __forceinline__ void backward8(const float* w, const float* x, const float* g, float r, float k, float* o, float* acc)
{
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        acc[j] = fmaf(w[j], x[j] * r, acc[j]);
        o[j] = fmaf(r, w[j] * g[j] - x[j] * k, o[j]);
    }
}

/* A warp per row, eight rows a block at a time. */
template <typename T>
__global__ void __launch_bounds__(256, 4)
decxb_rmsnorm_backward_kernel(const NormBwdArgs a)
{
    __shared__ float sums[8][256];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cols = (int)a.cols, first = lane * 8, count = min(8, cols - first);
    float acc[8] = {}, g[8];
    start_after_previous();
    load8_any(a.gamma, a.gamma_type, first, count, a.gvec, g);
    for (int64_t row = (int64_t)blockIdx.x * 8 + warp; row < a.rows; row += (int64_t)gridDim.x * 8) {
        float w[8], x[8], o[8];
        load8(static_cast<const T*>(a.dy) + row * a.lddy + first, count, a.vec, w);
        load8(static_cast<const T*>(a.h) + row * a.ldh + first, count, a.vec, x);
        load8(static_cast<const T*>(a.dr) + row * a.lddr + first, a.dr ? count : 0, a.vec, o);
        float sq = 0.0f, dot = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) { sq = fmaf(x[j], x[j], sq); dot = fmaf(w[j] * g[j], x[j], dot); }
        const float r = rsqrtf(warp_sum(sq) / (float)cols + a.eps), k = r * r * (warp_sum(dot) / (float)cols);
        backward8(w, x, g, r, k, o, acc);
        if (count > 0) store8(static_cast<T*>(a.dx) + row * a.lddx + first, count, a.vec, o);
    }
    if (!a.part) return;
    *reinterpret_cast<float4*>(&sums[warp][first]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
    *reinterpret_cast<float4*>(&sums[warp][first + 4]) = make_float4(acc[4], acc[5], acc[6], acc[7]);
    __syncthreads();
    if (const int c = threadIdx.x; c < cols) {
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) s += sums[w][c];
        a.part[(int64_t)blockIdx.x * cols + c] = s;
    }
}

/* A block per row, its rows arriving in shared memory by bulk copies `stages` rows ahead: a row is a chain of load, sum over
 * the block, store, and without the copies a block would have nothing on the way during most of it (8192 x 4096 bf16:
 * 122 us with loads into registers, 47.8 so, 5.6 TB/s). */
template <typename T, int VPT>
__global__ void __launch_bounds__(512, VPT == 1 ? 2 : 1)
decxb_rmsnorm_backward_rows_kernel(const NormBwdArgs a, const int stages, const Waits waits)
{
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float2 buf[2][17];              /* [16]: not 0 where a thread gave its wait up */
    __shared__ __align__(8) uint64_t bars[8];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, nwarps = blockDim.x >> 5, cols = (int)a.cols;
    const int arrays = a.dr ? 3 : 2;
    const uint32_t row_bytes = (uint32_t)cols * (uint32_t)sizeof(T);
    auto first = [&](int i) { return (i * (int)blockDim.x + tid) * 8; };
    auto fetch = [&](int64_t row, int st) {
        const uint32_t bar = tcptx::smem_u32(&bars[st]), at = tcptx::smem_u32(smem) + (uint32_t)(st * arrays) * row_bytes;
        tcptx::mbar_arrive_expect_tx(bar, row_bytes * arrays);
        if (row == waits.lost) return;
        bulk_load(at, static_cast<const T*>(a.dy) + row * a.lddy, row_bytes, bar);
        bulk_load(at + row_bytes, static_cast<const T*>(a.h) + row * a.ldh, row_bytes, bar);
        if (a.dr) bulk_load(at + 2 * row_bytes, static_cast<const T*>(a.dr) + row * a.lddr, row_bytes, bar);
    };
    if (tid == 0) {
        buf[0][16].x = buf[1][16].x = 0.0f;
        for (int st = 0; st < stages; ++st) tcptx::mbar_init(tcptx::smem_u32(&bars[st]), 1);
        tcptx::fence_barrier_init();
    }
    __syncthreads();
    start_after_previous();
    if (tid == 0)
        for (int st = 0; st < stages; ++st)
            if (blockIdx.x + (int64_t)st * gridDim.x < a.rows) fetch(blockIdx.x + (int64_t)st * gridDim.x, st);
    constexpr bool KEEP = VPT < 4;            /* gamma in registers; with four vectors a thread it is read again every row */
    float acc[VPT][8], g[KEEP ? VPT : 1][8];
    auto gamma = [&](int i) -> const float* {
        if constexpr (KEEP) return g[i];
        else { load8_any(a.gamma, a.gamma_type, first(i), cols - first(i), true, g[0]); return g[0]; }
    };
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        if constexpr (KEEP) load8_any(a.gamma, a.gamma_type, first(i), cols - first(i), true, g[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] = 0.0f;
    }
    int st = 0, turn = 0; uint32_t phase = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
        if (!wait_copy(tcptx::smem_u32(&bars[st]), phase, waits)) buf[turn][16].x = 1.0f;
        const T* in = reinterpret_cast<const T*>(smem + (size_t)(st * arrays) * row_bytes);
        Raw8<T> rw[VPT], rx[VPT], ro[VPT];
        float sq = 0.0f, dot = 0.0f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int n = first(i) < cols ? 8 : 0;
            load_raw(in + first(i), n, true, rw[i]);
            load_raw(in + cols + first(i), n, true, rx[i]);
            load_raw(in + 2 * cols + first(i), a.dr ? n : 0, true, ro[i]);
            float w[8], x[8];
            unpack(rw[i], w); unpack(rx[i], x);
            const float* gi = gamma(i);
#pragma unroll
            for (int j = 0; j < 8; ++j) { sq = fmaf(x[j], x[j], sq); dot = fmaf(w[j] * gi[j], x[j], dot); }
        }
        /* behind the barrier in here every thread has its values: the stage can be filled again */
        const float2 s = block_sum2(sq, dot, buf[turn], warp, lane, nwarps);
        const bool gone = buf[turn][16].x != 0.0f;
        if (tid == 0 && !gone && row + (int64_t)stages * gridDim.x < a.rows) fetch(row + (int64_t)stages * gridDim.x, st);
        const float r = rsqrtf(s.x / (float)cols + a.eps), k = r * r * (s.y / (float)cols);
        if (gone) {                            /* the row did not come: it and those behind it stay unwritten and out of dgamma */
            if (tid == 0) drain_copies(bars, stages, st, phase, row, a.rows);
            break;
        }
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            float w[8], x[8], o[8];
            unpack(rw[i], w); unpack(rx[i], x); unpack(ro[i], o);
            backward8(w, x, gamma(i), r, k, o, acc[i]);
            if (first(i) < cols) store8(static_cast<T*>(a.dx) + row * a.lddx + first(i), 8, true, o);
        }
        if (++st == stages) { st = 0; phase ^= 1u; }
    }
    if (!a.part) return;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
        if (first(i) < cols) store8(a.part + (int64_t)blockIdx.x * cols + first(i), 8, true, acc[i]);
}

/* Rows too long for that, or not aligned for it: each row is read twice and the sums for dgamma live in the workspace. */
template <typename T>
__global__ void __launch_bounds__(512)
decxb_rmsnorm_backward_wide_kernel(const NormBwdArgs a)
{
    __shared__ float2 buf[2][32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, nwarps = blockDim.x >> 5;
    start_after_previous();
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
        const T* dy = static_cast<const T*>(a.dy) + row * a.lddy;
        const T* h = static_cast<const T*>(a.h) + row * a.ldh;
        float sq = 0.0f, dot = 0.0f, w[8], x[8], g[8], o[8];
        for (int64_t c = (int64_t)tid * 8; c < a.cols; c += (int64_t)blockDim.x * 8) {
            const int n = (int)min((int64_t)8, a.cols - c);
            load8(dy + c, n, a.vec, w); load8(h + c, n, a.vec, x); load8_any(a.gamma, a.gamma_type, c, n, a.gvec, g);
#pragma unroll
            for (int j = 0; j < 8; ++j) { sq = fmaf(x[j], x[j], sq); dot = fmaf(w[j] * g[j], x[j], dot); }
        }
        const float2 s = block_sum2(sq, dot, buf[turn], warp, lane, nwarps);
        const float r = rsqrtf(s.x / (float)a.cols + a.eps);
        const float k = r * r * (s.y / (float)a.cols);
        for (int64_t c = (int64_t)tid * 8; c < a.cols; c += (int64_t)blockDim.x * 8) {
            const int n = (int)min((int64_t)8, a.cols - c);
            load8(dy + c, n, a.vec, w); load8(h + c, n, a.vec, x); load8_any(a.gamma, a.gamma_type, c, n, a.gvec, g);
            if (a.dr) load8(static_cast<const T*>(a.dr) + row * a.lddr + c, n, a.vec, o);
            else {
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j] = 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = fmaf(r, w[j] * g[j] - x[j] * k, o[j]);
            if (a.part) {
                float* p = a.part + (int64_t)blockIdx.x * a.cols + c;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j < n) p[j] = fmaf(w[j], x[j] * r, row == (int64_t)blockIdx.x ? 0.0f : p[j]);
            }
            store8(static_cast<T*>(a.dx) + row * a.lddx + c, n, a.vec, o);
        }
    }
}

/* dgamma[c] = sum over the workspace's rows: 32 columns a block, 32 groups of rows side by side. */
__global__ void __launch_bounds__(1024)
decxb_column_sum_kernel(const float* part, int parts, int64_t cols, float* out)
{
    __shared__ float sums[32][33];
    const int lane = threadIdx.x & 31, group = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    start_after_previous();
    float v = 0.0f;
    if (c < cols)
        for (int p = group; p < parts; p += 32) v += part[(int64_t)p * cols + c];
    sums[group][lane] = v;
    __syncthreads();
    v = warp_sum(sums[lane][group]);            /* warp g adds the 32 groups of column g */
    const int64_t co = (int64_t)blockIdx.x * 32 + group;
    if (lane == 0 && co < cols) out[co] = v;
}

/* Blocks to an SM, whose sums are the rows of the workspace: more of them where rows are short and a block's chain of load,
 * sum and store has little to move (16384 x 1024: 2 blocks and a warp a row 101 us).  From 4097 to 8192 columns two are planned and
 * the kernel's 122 registers let one on at a time; the other's shared memory is what fp32 rows of 4696 columns and more (three arrays; 7048,
 * two) lack for a second stage, so that those take the kernel that reads rows twice. */
constexpr int64_t WARP_COLS = 256;
int64_t backward_per_sm(int64_t cols) { return cols <= WARP_COLS ? 4 : cols <= 1024 ? 8 : cols <= 2048 ? 4 : cols <= 8192 ? 2 : 1; }
int64_t backward_blocks(const decxb_ctx* ctx, int64_t rows, int64_t cols)
{
    const int64_t most = ctx->sm_count * backward_per_sm(cols), have = cols <= WARP_COLS ? decxb_ceil_div(rows, 8) : rows;
    return have < most ? have : most;
}

template <typename T, int VPT>
int launch_backward_rows(decxb_ctx* ctx, const NormBwdArgs& a, unsigned grid, int stages, size_t smem, cudaStream_t s)
{
    auto kernel = decxb_rmsnorm_backward_rows_kernel<T, VPT>;
    static std::once_flag once[DECXB_MAX_DEVICES];
    static cudaError_t err[DECXB_MAX_DEVICES];
    std::call_once(once[ctx->device], [&] { err[ctx->device] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 225 * 1024); });
    if (err[ctx->device] != cudaSuccess) return decxb_fail(ctx, DECXB_ERR_CUDA, std::string("norm kernel attributes: ") + cudaGetErrorString(err[ctx->device]));
    return launch_after(ctx, kernel, grid, threads_for(decxb_ceil_div(a.cols, 8), VPT, 512), smem, s, a, stages, waits_of(ctx));
}

template <typename T>
int launch_norm_backward(decxb_ctx* ctx, const NormBwdArgs& a, float* dgamma, cudaStream_t s)
{
    const int64_t nvec = decxb_ceil_div(a.cols, 8), grid = backward_blocks(ctx, a.rows, a.cols);
    const int64_t row_bytes = a.cols * (int64_t)sizeof(T) * (a.dr ? 3 : 2);
    int64_t stages = 220 * 1024 / backward_per_sm(a.cols) / row_bytes;       /* rows of a block in shared memory */
    if (stages > 4) stages = 4;
    int rc;
    if (a.cols <= WARP_COLS) rc = launch_after(ctx, decxb_rmsnorm_backward_kernel<T>, (unsigned)grid, 256, 0, s, a);
    else if (a.vec && a.gvec && a.cols % 8 == 0 && nvec <= 2048 && stages >= 2)
        rc = nvec <= 512  ? launch_backward_rows<T, 1>(ctx, a, (unsigned)grid, (int)stages, (size_t)(stages * row_bytes), s)
           : nvec <= 1024 ? launch_backward_rows<T, 2>(ctx, a, (unsigned)grid, (int)stages, (size_t)(stages * row_bytes), s)
                          : launch_backward_rows<T, 4>(ctx, a, (unsigned)grid, (int)stages, (size_t)(stages * row_bytes), s);
    else
        rc = launch_after(ctx, decxb_rmsnorm_backward_wide_kernel<T>, (unsigned)grid, 512, 0, s, a);
    if (rc == DECXB_OK && dgamma)
        rc = launch_after(ctx, decxb_column_sum_kernel, (unsigned)decxb_ceil_div(a.cols, 32), 1024, 0, s, (const float*)a.part, (int)grid, a.cols, dgamma);
    return rc;
}

/* ---- quantisation -------------------------------------------------------------------------
 * A block of 256 threads holds one 128 x 128 tile of X in registers: thread (g, t) = (tid / 16, tid % 16) has rows
 * 8 g .. 8 g + 7 of columns 8 t .. 8 t + 7.  A row's 128 values lie in the 16 lanes of half a warp; a column's in
 * the 16 groups, which meet through shared memory.  The transposed codes leave through shared memory as well,
 * eight rows (8 bytes) of a column at a time, the 8-byte pieces of a column XOR-ed with the column group so that
 * the 16 lanes of a store fall into 16 different bank pairs.
 * 8192 x 4096 bf16 both ways takes 26.4 us (5.1 TB/s), one way 16.6 (6.0): 14.5 instructions an element of both, which is
 * about as long as the memory needs.  Blocks that stay and fetch the next tile while they code one were slower (35 us):
 * the reads that run ahead get in the way of the writes. */
struct QuantArgs {
    int64_t rows, cols, ldx;
    const void* x;
    int rule; bool vec;
    bool plain;                       /* x, q and t take vectors, 128 rows of each within 2 GiB            */
    int64_t tiles_c;
    struct Out { uint8_t* data; float* s; int64_t ld, srs, sbs; int type, block_rows; bool vec; } q, t;
};

/* Larger magnitude of two floats, or of two pairs of 16-bit numbers, NaN winning; the sign of the result means nothing. */
__device__ __forceinline__ uint32_t max_word(uint32_t a, uint32_t b, const __nv_bfloat16*)
{
    uint32_t r; asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r;
}
__device__ __forceinline__ uint32_t max_word(uint32_t a, uint32_t b, const __half*)
{
    uint32_t r; asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r;
}
__device__ __forceinline__ uint32_t max_word(uint32_t a, uint32_t b, const float*)
{
    float r; asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(__uint_as_float(a)), "f"(__uint_as_float(b))); return __float_as_uint(r);
}
template <typename T>
__device__ __forceinline__ uint32_t shuffle_max(uint32_t a, int o)
{
    return max_word(a, __shfl_xor_sync(0xffffffffu, a, o), static_cast<const T*>(nullptr));
}

/* W words hold the eight columns of a row, E columns to a word; magnitudes are compared as words, two columns of 16 bits at once. */
template <typename T>
struct QuantShared {
    static constexpr int W = 2 * (int)sizeof(T), E = 8 / W;
    uint32_t colmax[8][16 * W];
    uint32_t wmax[8];
    alignas(16) Quantiser colq[128];
    alignas(16) uint8_t tr[128 * 128];
};

/* WHOLE: 128 rows and columns there, every row a vector of its own, and the tile's rows within 2 GiB of one another (with the
 * questions and the 64-bit addresses of the general case half as many instructions again: 32 us for 26.4). */
template <typename T, int TYPE, bool WHOLE>
__device__ __forceinline__ void quantize_tile(const QuantArgs& a, QuantShared<T>& sh, int64_t tile_r, int64_t tile_c)
{
    constexpr int W = QuantShared<T>::W, E = QuantShared<T>::E;
    constexpr uint32_t MAG = E == 2 ? 0x7fff7fffu : 0x7fffffffu;
    const T* const kind = nullptr;
    auto& colmax = sh.colmax; auto& wmax = sh.wmax; auto& colq = sh.colq; auto& tr = sh.tr;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = tid >> 4, t = tid & 15;
    const int64_t r0 = tile_r * 128, c0 = tile_c * 128;
    const int64_t row = r0 + g * 8, col = c0 + t * 8;
    const int nr = WHOLE ? 8 : (int)max((int64_t)0, min((int64_t)8, a.rows - row));          /* rows and columns that exist here */
    const int nc = WHOLE ? 8 : (int)max((int64_t)0, min((int64_t)8, a.cols - col));
    const bool full = WHOLE || c0 + 128 <= a.cols;
    Raw8<T> x[8];
    if constexpr (WHOLE) {
        const uint8_t* base = static_cast<const uint8_t*>(a.x) + (r0 * a.ldx + c0) * (int64_t)sizeof(T);
        const uint32_t pitch = (uint32_t)a.ldx * (uint32_t)sizeof(T);
        uint32_t at = (uint32_t)(g * 8) * pitch + (uint32_t)(t * 8 * (int)sizeof(T));
#pragma unroll
        for (int i = 0; i < 8; ++i, at += pitch)
#pragma unroll
            for (int k = 0; k < (int)sizeof(T) / 2; ++k) x[i].u[k] = *(reinterpret_cast<const uint4*>(base + at) + k);
    } else {
        const T* px = static_cast<const T*>(a.x) + row * a.ldx + col;
        if (full && a.vec) {
#pragma unroll
            for (int i = 0; i < 8; ++i, px += a.ldx)
#pragma unroll
                for (int k = 0; k < (int)sizeof(T) / 2; ++k) x[i].u[k] = i < nr ? *(reinterpret_cast<const uint4*>(px) + k) : make_uint4(0, 0, 0, 0);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i, px += a.ldx) load_raw(px, i < nr ? nc : 0, a.vec, x[i]);
        }
    }
    auto word = [&](int i, int k) { return reinterpret_cast<const uint32_t*>(x[i].u)[k]; };
    auto lane_of = [&](uint32_t w, int e) -> float {      /* column e of a word */
        if constexpr (E == 2) { float f, g; halves(w, kind, f, g); return e ? g : f; }
        else return __uint_as_float(w);
    };

    const bool whole = (a.q.data && a.q.block_rows == 128) || (a.t.data && a.t.block_rows == 128);
    const bool by_col = a.t.data && a.t.block_rows == 1;
    if (whole || by_col) {
        uint32_t m = 0;
#pragma unroll
        for (int k = 0; k < W; ++k) {
            uint32_t c = word(0, k);
#pragma unroll
            for (int i = 1; i < 8; ++i) c = max_word(c, word(i, k), kind);
            c = shuffle_max<T>(c, 16);
            if (by_col && lane < 16) colmax[warp][t * W + k] = c;
            m = k ? max_word(m, c, kind) : c;
        }
#pragma unroll
        for (int o = 8; o; o >>= 1) m = shuffle_max<T>(m, o);
        if (lane == 0) wmax[warp] = m;
        __syncthreads();
    }
    float tile_max = 0.0f;
    if (whole) {
        uint32_t m = wmax[0];
#pragma unroll
        for (int w = 1; w < 8; ++w) m = max_word(m, wmax[w], kind);
#pragma unroll
        for (int e = 0; e < E; ++e) tile_max = max_nan(tile_max, lane_of(m & MAG, e));
    }

    /* one thread a column makes the scales of the transpose's rows while the others go on */
    if (by_col && tid < 128) {
        uint32_t m = colmax[0][tid / E];
#pragma unroll
        for (int w = 1; w < 8; ++w) m = max_word(m, colmax[w][tid / E], kind);
        const float s = scale_of(lane_of(m & MAG, tid % E), TYPE, a.rule);
        if (c0 + tid < a.cols) a.t.s[(c0 + tid) * a.t.srs + tile_r * a.t.sbs] = s;
        colq[tid] = quantiser(s);
    }

    if (a.q.data) {
        float s = 0.0f;
        if (a.q.block_rows == 128) {
            s = scale_of(tile_max, TYPE, a.rule);
            if (tid == 0) a.q.s[tile_r * a.q.srs + tile_c * a.q.sbs] = s;
        } else {
            /* largest of each of the eight rows (16 bits: rows i and i + 4 in one word), halved over the lanes at every exchange:
             * lane t ends with row t / 2 */
            uint32_t f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                f[i] = word(i, 0);
#pragma unroll
                for (int k = 1; k < W; ++k) f[i] = max_word(f[i], word(i, k), kind);
            }
            if constexpr (E == 2) {
#pragma unroll
                for (int i = 0; i < 4; ++i) f[i] = max_word(__byte_perm(f[i], f[i + 4], 0x5410), __byte_perm(f[i], f[i + 4], 0x7632), kind);
            }
#pragma unroll
            for (int n = 4 / E; n; n >>= 1) {
                const bool up = t & (2 * n);
#pragma unroll
                for (int i = 0; i < n; ++i) {
                    const uint32_t keep = up ? f[n + i] : f[i], give = up ? f[i] : f[n + i];
                    f[i] = max_word(keep, __shfl_xor_sync(0xffffffffu, give, 2 * n), kind);
                }
            }
            if constexpr (E == 2) f[0] = shuffle_max<T>(f[0], 8);
            f[0] = shuffle_max<T>(f[0], 1) & MAG;
            s = scale_of(E == 2 && !(t & 8) ? lane_of(f[0], 0) : lane_of(f[0], E - 1), TYPE, a.rule);
            if ((t & 1) == 0 && (t >> 1) < nr) a.q.s[(row + (t >> 1)) * a.q.srs + tile_c * a.q.sbs] = s;
        }
        Quantiser z = quantiser(s);
        const float s_row = z.minus_s, inv_row = z.inv;
        uint8_t* q = a.q.data + (WHOLE ? r0 * a.q.ld + c0 : row * a.q.ld + col);
        uint32_t at = (uint32_t)(g * 8) * (uint32_t)a.q.ld + (uint32_t)(t * 8);
#pragma unroll
        for (int i = 0; i < 8; ++i, at += (uint32_t)a.q.ld) {
            if (a.q.block_rows == 1) {
                z.minus_s = __shfl_sync(0xffffffffu, s_row, 2 * i, 16);
                z.inv = __shfl_sync(0xffffffffu, inv_row, 2 * i, 16);
            }
            float v[8];
            unpack(x[i], v);
            const uint2 c = codes8<TYPE>(v, z);
            if constexpr (WHOLE) *reinterpret_cast<uint2*>(q + at) = c;
            else if (full && a.q.vec) { if (i < nr) *reinterpret_cast<uint2*>(q + i * a.q.ld) = c; }
            else if (i < nr && nc > 0) store_codes8(q + i * a.q.ld, nc, a.q.vec, c);
        }
    }

    if (a.t.data) {
        if (by_col) __syncthreads();
        const float st = a.t.block_rows == 128 ? scale_of(tile_max, TYPE, a.rule) : 0.0f;
        if (a.t.block_rows == 128 && tid == 0) a.t.s[tile_c * a.t.srs + tile_r * a.t.sbs] = st;
        Quantiser z = quantiser(st);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (by_col) z = colq[t * 8 + j];
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = lane_of(word(i, j / E), j % E);
            *reinterpret_cast<uint2*>(tr + (t * 8 + j) * 128 + ((g ^ t) << 3)) = codes8<TYPE>(v, z);
        }
        __syncthreads();
        /* out: row c of the transpose, eight of X's rows per thread, 16 lanes a row */
        const int nro = WHOLE ? 8 : (int)max((int64_t)0, min((int64_t)8, a.rows - (r0 + t * 8)));
        uint8_t* o = a.t.data + (WHOLE ? c0 * a.t.ld + r0 : (c0 + g) * a.t.ld + r0 + t * 8);
        uint32_t at = (uint32_t)g * (uint32_t)a.t.ld + (uint32_t)(t * 8);
#pragma unroll
        for (int p = 0; p < 8; ++p, at += 16 * (uint32_t)a.t.ld) {
            const int c = p * 16 + g;
            const uint2 k = *reinterpret_cast<const uint2*>(tr + c * 128 + ((t ^ (c >> 3)) << 3));
            if constexpr (WHOLE) *reinterpret_cast<uint2*>(o + at) = k;
            else if (c0 + c < a.cols && nro > 0) store_codes8(o + p * 16 * a.t.ld, nro, a.t.vec, k);
        }
    }
}

template <typename T, int TYPE>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 4 : 2)
decxb_quantize_fp8_kernel(const QuantArgs a)
{
    __shared__ QuantShared<T> sh;
    const int64_t tile_r = blockIdx.x / a.tiles_c, tile_c = blockIdx.x % a.tiles_c;
    start_after_previous();
    if (a.plain && tile_r * 128 + 128 <= a.rows && tile_c * 128 + 128 <= a.cols) quantize_tile<T, TYPE, true>(a, sh, tile_r, tile_c);
    else                                                                        quantize_tile<T, TYPE, false>(a, sh, tile_r, tile_c);
}

template <typename T>
int launch_quantize(decxb_ctx* ctx, const QuantArgs& a, cudaStream_t s)
{
    const int64_t tiles = decxb_ceil_div(a.rows, 128) * a.tiles_c;
    if (tiles > 0x7fffffffLL) return decxb_fail(ctx, DECXB_ERR_TOO_LARGE, "tiles of 128 x 128");
    return (a.q.data ? a.q.type : a.t.type) == DECXB_FP8_E4M3
        ? launch_after(ctx, decxb_quantize_fp8_kernel<T, DECXB_FP8_E4M3>, (unsigned)tiles, 256, 0, s, a)
        : launch_after(ctx, decxb_quantize_fp8_kernel<T, DECXB_FP8_E5M2>, (unsigned)tiles, 256, 0, s, a);
}

QuantArgs::Out out_of(const decxb_fp8_matrix* m)
{
    if (!m) return {};
    return {static_cast<uint8_t*>(m->data), m->scales, m->ld, m->scale_row_stride, m->scale_block_stride, m->type, m->block_rows,
            aligned(m->data, m->ld, 8)};
}

int quantize(decxb_ctx* ctx, int x_type, int64_t rows, int64_t cols, const void* X, int64_t ldx, int rule,
             const decxb_fp8_matrix* Q, const decxb_fp8_matrix* Qt, cudaStream_t s)
{
    if (!type_ok(x_type)) return decxb_fail(ctx, DECXB_ERR_BAD_FLAG, "x_type");
    if (rule != DECXB_SCALE_AMAX && rule != DECXB_SCALE_POW2) return decxb_fail(ctx, DECXB_ERR_BAD_FLAG, "scale rule");
    if (rows < 0 || cols < 0) return decxb_fail(ctx, DECXB_ERR_BAD_PARAM, "negative size");
    if (!Q && !Qt) return decxb_fail(ctx, DECXB_ERR_BAD_PARAM, "nothing to write");
    int rc;
    if (Q && (rc = check_output(ctx, Q, "Q", rows, cols))) return rc;
    if (Qt && (rc = check_output(ctx, Qt, "Qt", cols, rows))) return rc;
    if (rows == 0 || cols == 0) return DECXB_OK;
    if ((rc = check_array(ctx, X, ldx, cols, size_of(x_type), "X"))) return rc;
    if (Q && Qt && Q->type != Qt->type) {         /* one type a launch */
        rc = quantize(ctx, x_type, rows, cols, X, ldx, rule, Q, nullptr, s);
        return rc ? rc : quantize(ctx, x_type, rows, cols, X, ldx, rule, nullptr, Qt, s);
    }
    QuantArgs a = {};
    a.rows = rows; a.cols = cols; a.x = X; a.ldx = ldx; a.rule = rule;
    a.vec = aligned(X, ldx * size_of(x_type), 16);
    a.tiles_c = decxb_ceil_div(cols, 128);
    a.q = out_of(Q); a.t = out_of(Qt);
    constexpr int64_t NEAR = 1 << 24;             /* bytes of a row */
    a.plain = a.vec && ldx * size_of(x_type) < NEAR && (!Q || (a.q.vec && Q->ld < NEAR)) && (!Qt || (a.t.vec && Qt->ld < NEAR));
    if (x_type == DECXB_F32) return launch_quantize<float>(ctx, a, s);
    if (x_type == DECXB_F16) return launch_quantize<__half>(ctx, a, s);
    return launch_quantize<__nv_bfloat16>(ctx, a, s);
}

int norm_common(decxb_ctx* ctx, int type, int64_t rows, int64_t cols, int gamma_type, float eps)
{
    if (!type_ok(type) || !type_ok(gamma_type)) return decxb_fail(ctx, DECXB_ERR_BAD_FLAG, "type");
    if (rows < 0 || cols <= 0) return decxb_fail(ctx, DECXB_ERR_BAD_PARAM, "rows must not be negative, cols must be positive");
    if (rows > 0x7fffffffLL || cols > 0x7fffffffLL) return decxb_fail(ctx, DECXB_ERR_TOO_LARGE, "rows or cols");
    if (!(eps >= 0.0f) || eps > 3.0e38f) return decxb_fail(ctx, DECXB_ERR_BAD_PARAM, "eps must be a finite number >= 0");
    return DECXB_OK;
}

int norm(decxb_ctx* ctx, int type, int64_t rows, int64_t cols, const void* X, int64_t ldx, const void* R, int64_t ldr,
         const void* gamma, int gamma_type, float eps, void* H, int64_t ldh, void* Y, int64_t ldy, int rule,
         const decxb_fp8_matrix* Q, cudaStream_t s)
{
    int rc = norm_common(ctx, type, rows, cols, gamma_type, eps);
    if (rc) return rc;
    if (rule != DECXB_SCALE_AMAX && rule != DECXB_SCALE_POW2) return decxb_fail(ctx, DECXB_ERR_BAD_FLAG, "scale rule");
    if (!H && !Y && !Q) return decxb_fail(ctx, DECXB_ERR_BAD_PARAM, "nothing to write");
    if (Q && (rc = check_output(ctx, Q, "Q", rows, cols))) return rc;
    if (Q && Q->block_rows != 1) return decxb_fail(ctx, DECXB_ERR_BAD_PARAM, "Q: block_rows must be 1");
    if (rows == 0) return DECXB_OK;
    const int e = size_of(type);
    if ((rc = check_array(ctx, X, ldx, cols, e, "X")) || (rc = check_array(ctx, gamma, cols, cols, size_of(gamma_type), "gamma"))) return rc;
    if (R && (rc = check_array(ctx, R, ldr, cols, e, "R"))) return rc;
    if (H && (rc = check_array(ctx, H, ldh, cols, e, "H"))) return rc;
    if (Y && (rc = check_array(ctx, Y, ldy, cols, e, "Y"))) return rc;
    if (H && H == Y) return decxb_fail(ctx, DECXB_ERR_BAD_PARAM, "H and Y are the same array");
    if ((H == X && H && ldh != ldx) || (H == R && H && ldh != ldr) || (Y == X && Y && ldy != ldx) || (Y == R && Y && ldy != ldr))
        return decxb_fail(ctx, DECXB_ERR_BAD_PARAM, "an output in place of an input needs its leading dimension");
    NormArgs a = {};
    a.rows = rows; a.cols = cols; a.x = X; a.r = R; a.gamma = gamma; a.h = H; a.y = Y;
    a.ldx = ldx; a.ldr = ldr; a.ldh = ldh; a.ldy = ldy; a.gamma_type = gamma_type; a.rule = rule; a.eps = eps;
    a.vec = aligned(X, ldx * e, 16) && (!R || aligned(R, ldr * e, 16)) && (!H || aligned(H, ldh * e, 16)) && (!Y || aligned(Y, ldy * e, 16));
    a.gvec = aligned(gamma, 0, 16);
    if (Q) {
        a.q = static_cast<uint8_t*>(Q->data); a.ldq = Q->ld; a.s = Q->scales; a.srs = Q->scale_row_stride; a.sbs = Q->scale_block_stride;
        a.qtype = Q->type; a.qvec = aligned(Q->data, Q->ld, 8);
    }
    if (type == DECXB_F32) return launch_norm<float>(ctx, a, s);
    if (type == DECXB_F16) return launch_norm<__half>(ctx, a, s);
    return launch_norm<__nv_bfloat16>(ctx, a, s);
}

size_t backward_bytes(const decxb_ctx* ctx, int64_t rows, int64_t cols)
{
    return (size_t)backward_blocks(ctx, rows, cols) * (size_t)cols * sizeof(float);
}

int norm_backward(decxb_ctx* ctx, int type, int64_t rows, int64_t cols, const void* dY, int64_t lddy, const void* H, int64_t ldh,
                  const void* gamma, int gamma_type, float eps, const void* dR, int64_t lddr, void* dX, int64_t lddx, float* dgamma,
                  void* workspace, size_t workspace_bytes, cudaStream_t s)
{
    int rc = norm_common(ctx, type, rows, cols, gamma_type, eps);
    if (rc) return rc;
    if (reinterpret_cast<uintptr_t>(dgamma) % 4) return decxb_fail(ctx, DECXB_ERR_BAD_PARAM, "dgamma: not aligned to its elements");
    if (rows == 0) {
        if (dgamma) DECXB_CUDA_TRY(ctx, cudaMemsetAsync(dgamma, 0, (size_t)cols * sizeof(float), s));
        return DECXB_OK;
    }
    const int e = size_of(type);
    if ((rc = check_array(ctx, dY, lddy, cols, e, "dY")) || (rc = check_array(ctx, H, ldh, cols, e, "H")) ||
        (rc = check_array(ctx, gamma, cols, cols, size_of(gamma_type), "gamma")) || (rc = check_array(ctx, dX, lddx, cols, e, "dX"))) return rc;
    if (dR && (rc = check_array(ctx, dR, lddr, cols, e, "dR"))) return rc;
    if ((dX == dY && lddx != lddy) || (dX == dR && lddx != lddr))
        return decxb_fail(ctx, DECXB_ERR_BAD_PARAM, "dX in place of an input needs its leading dimension");
    if (dX == H) return decxb_fail(ctx, DECXB_ERR_BAD_PARAM, "dX may not be H");
    const size_t need = dgamma ? backward_bytes(ctx, rows, cols) : 0;
    NormBwdArgs a = {};
    a.rows = rows; a.cols = cols; a.dy = dY; a.h = H; a.dr = dR; a.gamma = gamma; a.dx = dX;
    a.lddy = lddy; a.ldh = ldh; a.lddr = lddr; a.lddx = lddx; a.gamma_type = gamma_type; a.eps = eps;
    a.vec = aligned(dY, lddy * e, 16) && aligned(H, ldh * e, 16) && (!dR || aligned(dR, lddr * e, 16)) && aligned(dX, lddx * e, 16);
    a.gvec = aligned(gamma, 0, 16);
    void* scratch = nullptr;
    if (need && workspace) {
        if (workspace_bytes < need) return decxb_fail(ctx, DECXB_ERR_BAD_PARAM, "workspace of " + std::to_string(need) + " bytes needed");
        if (reinterpret_cast<uintptr_t>(workspace) % 16) return decxb_fail(ctx, DECXB_ERR_BAD_PARAM, "workspace not 16-byte aligned");
        a.part = static_cast<float*>(workspace);
    } else if (need) {
        if ((rc = refuse_capture(ctx, s, "no workspace was given"))) return rc;
        if ((rc = decxb_malloc_on_stream(ctx, need, &scratch, s))) return rc;
        a.part = static_cast<float*>(scratch);
    }
    rc = type == DECXB_F32 ? launch_norm_backward<float>(ctx, a, dgamma, s)
       : type == DECXB_F16 ? launch_norm_backward<__half>(ctx, a, dgamma, s)
                           : launch_norm_backward<__nv_bfloat16>(ctx, a, dgamma, s);
    if (scratch) decxb_free_on_stream(ctx, scratch, s);
    return rc;
}

cudaStream_t stream_of(decxb_ctx* ctx, void* stream) { return stream ? (cudaStream_t)stream : ctx->stream; }

}  // namespace

extern "C" int decxb_quantize_fp8(decxb_ctx* ctx, int x_type, int64_t rows, int64_t cols, const void* X, int64_t ldx,
                                  int scale_rule, const decxb_fp8_matrix* Q, const decxb_fp8_matrix* Qt, void* stream)
try {
    DeviceScope dev(ctx);
    if (dev.status) return dev.status;
    return quantize(ctx, x_type, rows, cols, X, ldx, scale_rule, Q, Qt, stream_of(ctx, stream));
} catch (...) { return DECXB_ERR_ALLOC; }      /* the host's memory, or a lock of the runtime */

extern "C" int decxb_rmsnorm(decxb_ctx* ctx, int type, int64_t rows, int64_t cols, const void* X, int64_t ldx,
                             const void* R, int64_t ldr, const void* gamma, int gamma_type, float eps,
                             void* H, int64_t ldh, void* Y, int64_t ldy,
                             int scale_rule, const decxb_fp8_matrix* Q, void* stream)
try {
    DeviceScope dev(ctx);
    if (dev.status) return dev.status;
    return norm(ctx, type, rows, cols, X, ldx, R, ldr, gamma, gamma_type, eps, H, ldh, Y, ldy, scale_rule, Q, stream_of(ctx, stream));
} catch (...) { return DECXB_ERR_ALLOC; }      /* the host's memory, or a lock of the runtime */

extern "C" int decxb_rmsnorm_backward_workspace(decxb_ctx* ctx, int64_t rows, int64_t cols, size_t* bytes)
{
    if (!ctx || ctx->device < 0) return DECXB_ERR_NOT_INIT;
    if (!bytes || rows < 0 || cols < 0) return DECXB_ERR_BAD_PARAM;
    *bytes = backward_bytes(ctx, rows, cols);
    return DECXB_OK;
}

extern "C" int decxb_rmsnorm_backward(decxb_ctx* ctx, int type, int64_t rows, int64_t cols,
                                      const void* dY, int64_t lddy, const void* H, int64_t ldh,
                                      const void* gamma, int gamma_type, float eps,
                                      const void* dR, int64_t lddr, void* dX, int64_t lddx, float* dgamma,
                                      void* workspace, size_t workspace_bytes, void* stream)
try {
    DeviceScope dev(ctx);
    if (dev.status) return dev.status;
    return norm_backward(ctx, type, rows, cols, dY, lddy, H, ldh, gamma, gamma_type, eps, dR, lddr, dX, lddx, dgamma, workspace,
                         workspace_bytes, stream_of(ctx, stream));
} catch (...) { return DECXB_ERR_ALLOC; }      /* the host's memory, or a lock of the runtime */
