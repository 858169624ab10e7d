/* Shared by the 8-bit linear layer's kernels: element types, 8-element vectors, fp8 codes and scales, argument checks. */
#ifndef DECXB_FP8_CUH_
#define DECXB_FP8_CUH_

#include "common.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace fp8 {

/* ------------------------------------------------------------------ elements --------- */
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

/* The two elements of a 32-bit word as floats (bf16: one instruction each, where a conversion of the halves takes two). */
__device__ __forceinline__ void halves(uint32_t w, const __nv_bfloat16*, float& a, float& b)
{
    a = __uint_as_float(w << 16); b = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ void halves(uint32_t w, const __half*, float& a, float& b)
{
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    a = f.x; b = f.y;
}
template <typename T>
__device__ __forceinline__ void unpack4(const uint4& u, float* v)
{
    const T* const kind = nullptr;
    halves(u.x, kind, v[0], v[1]); halves(u.y, kind, v[2], v[3]); halves(u.z, kind, v[4], v[5]); halves(u.w, kind, v[6], v[7]);
}

/* Eight consecutive elements of a row as floats.  `n` of them exist (the others read as 0); `vec`: the
 * address is 16-byte aligned, so a whole vector moves in 128-bit accesses. */
template <typename T>
__device__ __forceinline__ void load8(const T* p, int n, bool vec, float* v)
{
    if (n >= 8 && vec) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = *reinterpret_cast<const float4*>(p), b = *(reinterpret_cast<const float4*>(p) + 1);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            unpack4<T>(*reinterpret_cast<const uint4*>(p), v);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < n ? to_f32(p[j]) : 0.0f;
    }
}

/* Eight elements as they lie in memory: what a thread keeps of a row until it needs the values. */
template <typename T> struct Raw8 { uint4 u[sizeof(T) / 2]; };
template <typename T>
__device__ __forceinline__ void load_raw(const T* p, int n, bool vec, Raw8<T>& o)
{
    if (n >= 8 && vec) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) o.u[i] = *(reinterpret_cast<const uint4*>(p) + i);
    } else {
        T* e = reinterpret_cast<T*>(o.u);
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = j < n ? p[j] : from_f32<T>(0.0f);
    }
}
template <typename T>
__device__ __forceinline__ void unpack(const Raw8<T>& r, float* v)
{
    if constexpr (sizeof(T) == 2) unpack4<T>(r.u[0], v);
    else {
        const float* e = reinterpret_cast<const float*>(r.u);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = e[j];
    }
}

__device__ __forceinline__ uint32_t joined(float a, float b, const __nv_bfloat16*)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t joined(float a, float b, const __half*)
{
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, int n, bool vec, const float* v)
{
    if (n >= 8 && vec) {
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
            *(reinterpret_cast<float4*>(p) + 1) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            const T* const kind = nullptr;
            *reinterpret_cast<uint4*>(p) = make_uint4(joined(v[0], v[1], kind), joined(v[2], v[3], kind), joined(v[4], v[5], kind), joined(v[6], v[7], kind));
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) if (j < n) p[j] = from_f32<T>(v[j]);
    }
}

/* The same for gamma, whose type is the call's own choice (uniform branch). */
__device__ __forceinline__ void load8_any(const void* base, int type, int64_t at, int n, bool vec, float* v)
{
    if (type == DECXB_F32)      load8(static_cast<const float*>(base) + at, n, vec, v);
    else if (type == DECXB_F16) load8(static_cast<const __half*>(base) + at, n, vec, v);
    else                        load8(static_cast<const __nv_bfloat16*>(base) + at, n, vec, v);
}

/* Two fp32 numbers an instruction (the rate of the arithmetic is the same, that of issuing is not). */
__device__ __forceinline__ uint64_t pack2(float a, float b) { uint64_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) { uint64_t r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r;
}

/* ------------------------------------------------------------------ codes and scales -- */
/* NaN wins (fmaxf would drop it): a NaN in a block has to reach its scale. */
__device__ __forceinline__ float max_nan(float a, float b)
{
    float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r;
}

/* amax / largest value, correctly rounded (a product with the reciprocal and one correction by the remainder, Markstein's
 * method), then the rule; infinity and NaN pass. */
__device__ __forceinline__ float scale_of(float amax, int type, int rule)
{
    const float most = type == DECXB_FP8_E4M3 ? 448.0f : 57344.0f, inv = type == DECXB_FP8_E4M3 ? 1.0f / 448.0f : 1.0f / 57344.0f;
    const float q = amax * inv;
    float s = amax < INFINITY ? fmaf(fmaf(-q, most, amax), inv, q) : amax;
    if (rule == DECXB_SCALE_POW2) {
        /* up to the next power of two: exponent + 1 unless the mantissa is zero (infinity and NaN stay) */
        const uint32_t u = __float_as_uint(s);
        if ((u & 0x7f800000u) != 0x7f800000u && (u & 0x007fffffu)) s = __uint_as_float((u & 0x7f800000u) + 0x00800000u);
    }
    return s < 1.17549435e-38f ? 1.17549435e-38f : s;
}

/* What a block's scale does to its values.  With the amax rule x / s of 16-bit x often lies half way between two codes but for
 * the rounding of s itself, so a product with 1 / s alone, one step of fp32 off, turns four codes in ten thousand
 * over: one correction by the remainder x - q s (Markstein's) makes it the fp32 quotient.  (With the power-of-two rule the product is
 * exact and the remainder 0.) */
struct alignas(8) Quantiser { float inv, minus_s; };    /* 1 / scale, and -scale (0 for an infinite one, whose finite values give 0) */
__device__ __forceinline__ Quantiser quantiser(float scale)
{
    return Quantiser{__frcp_rn(scale), scale < INFINITY ? -scale : 0.0f};
}

template <int TYPE>
__device__ __forceinline__ uint32_t codes4(const float* f)
{
    uint32_t r;
    if constexpr (TYPE == DECXB_FP8_E4M3)
        asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\tmov.b32 %0, {lo, hi};\n\t}"
            : "=r"(r) : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]));
    else
        asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e5m2x2.f32 lo, %2, %1;\n\tcvt.rn.satfinite.e5m2x2.f32 hi, %4, %3;\n\tmov.b32 %0, {lo, hi};\n\t}"
            : "=r"(r) : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]));
    return r;
}

/* Eight codes, rounded to nearest even; saturation only meets what the scale's own rounding pushed a hair over the
 * largest value. */
template <int TYPE>
__device__ __forceinline__ uint2 codes8(const float* v, const Quantiser& z)
{
    const uint64_t inv = pack2(z.inv, z.inv), s = pack2(z.minus_s, z.minus_s);
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const uint64_t x = pack2(v[j], v[j + 1]), q = mul2(x, inv);
        unpack2(fma2(fma2(q, s, x), inv, q), f[j], f[j + 1]);
    }
    return make_uint2(codes4<TYPE>(f), codes4<TYPE>(f + 4));
}

__device__ __forceinline__ void store_codes8(uint8_t* p, int n, bool vec, uint2 c)
{
    if (n >= 8 && vec) *reinterpret_cast<uint2*>(p) = c;
    else {
#pragma unroll 1
        for (int j = 0; j < n && j < 8; ++j) p[j] = (uint8_t)((j < 4 ? c.x : c.y) >> (8 * (j & 3)));
    }
}

/* ------------------------------------------------------------------ waits ------------ */
/* What a launch's waits go by.  A wait that lasts longer than the limit gives up, and the launch's other waits with it; those of other
 * launches do not, since what they wait for may well come. */
struct Waits {
    decxb_dev_status* status;
    long long limit_ns;
    uint32_t launch;                  /* this launch's number, not 0                         */
    int64_t lost;                     /* row or tile whose copies are left out (tests; -1: none) */
};
__device__ __forceinline__ bool gave_up(const Waits& w) { return *reinterpret_cast<volatile uint32_t*>(&w.status->launch) == w.launch; }
__device__ __forceinline__ void give_up(const Waits& w, int where, int detail)
{
    if (atomicCAS(&w.status->code, 0, DECXB_DEVERR_WAIT_EXPIRED) == 0) {
        w.status->where = where; w.status->block = (int)blockIdx.x; w.status->detail = detail;
    }
    *reinterpret_cast<volatile uint32_t*>(&w.status->launch) = w.launch;
    __threadfence_system();
}

/* ------------------------------------------------------------------ host side -------- */
/* Makes the context's device current for one entry and puts the caller's back. */
struct DeviceScope {
    int prev = -1, status;
    explicit DeviceScope(decxb_ctx* ctx)
    {
        if (cudaGetDevice(&prev) != cudaSuccess) { cudaGetLastError(); prev = -1; }
        status = decxb_bind(ctx);
        if (ctx && prev == ctx->device) prev = -1;
    }
    ~DeviceScope() { if (prev >= 0) cudaSetDevice(prev); }
};

inline int size_of(int type) { return type == DECXB_F32 ? 4 : 2; }
inline bool type_ok(int type) { return type == DECXB_F32 || type == DECXB_F16 || type == DECXB_BF16; }
inline bool aligned(const void* p, int64_t row_bytes, int to) { return (reinterpret_cast<uintptr_t>(p) % to) == 0 && row_bytes % to == 0; }

/* An fp8 matrix as an argument: `rows` x `cols` (-1: any). */
inline int check_matrix(decxb_ctx* ctx, const decxb_fp8_matrix* m, const char* name, int64_t rows, int64_t cols)
{
    const std::string n(name);
    if (m->type != DECXB_FP8_E4M3 && m->type != DECXB_FP8_E5M2) return decxb_fail(ctx, DECXB_ERR_BAD_FLAG, n + ": fp8 type");
    if (m->block_rows != 1 && m->block_rows != 128) return decxb_fail(ctx, DECXB_ERR_BAD_PARAM, n + ": block_rows must be 1 or 128");
    if (m->rows < 0 || m->cols < 0) return decxb_fail(ctx, DECXB_ERR_BAD_PARAM, n + ": negative size");
    if ((rows >= 0 && m->rows != rows) || (cols >= 0 && m->cols != cols)) return decxb_fail(ctx, DECXB_ERR_DIM_MISMATCH, n + ": rows or cols");
    if (m->ld < m->cols) return decxb_fail(ctx, DECXB_ERR_DIM_MISMATCH, n + ": leading dimension smaller than the row length");
    if (m->rows > 0x7fffffffLL || m->cols > 0x7fffffffLL) return decxb_fail(ctx, DECXB_ERR_TOO_LARGE, n + ": rows or cols");
    if (m->scale_row_stride < 0 || m->scale_block_stride < 0) return decxb_fail(ctx, DECXB_ERR_BAD_PARAM, n + ": negative scale stride");
    if (m->rows > 0 && m->cols > 0 && (!m->data || !m->scales)) return decxb_fail(ctx, DECXB_ERR_BAD_PARAM, n + ": null data or scales");
    if (reinterpret_cast<uintptr_t>(m->scales) % 4) return decxb_fail(ctx, DECXB_ERR_BAD_PARAM, n + ": scales not 4-byte aligned");
    return DECXB_OK;
}

/* As an output: its scales may not share words either. */
inline int check_output(decxb_ctx* ctx, const decxb_fp8_matrix* m, const char* name, int64_t rows, int64_t cols)
{
    if (int rc = check_matrix(ctx, m, name, rows, cols)) return rc;
    const int64_t r = decxb_ceil_div(m->rows, m->block_rows), c = decxb_ceil_div(m->cols, 128);
    const int64_t a = m->scale_row_stride, b = m->scale_block_stride;
    const bool apart = (r <= 1 || c <= 1) ? !((r > 1 && a == 0) || (c > 1 && b == 0)) : (b > 0 && a > (c - 1) * b) || (a > 0 && b > (r - 1) * a);
    if (!apart) return decxb_fail(ctx, DECXB_ERR_BAD_PARAM, std::string(name) + ": scale strides make blocks share a scale");
    return DECXB_OK;
}

/* A [rows][cols] array argument of element size `e`. */
inline int check_array(decxb_ctx* ctx, const void* p, int64_t ld, int64_t cols, int e, const char* name)
{
    if (!p) return decxb_fail(ctx, DECXB_ERR_BAD_PARAM, std::string(name) + ": null");
    if (reinterpret_cast<uintptr_t>(p) % e) return decxb_fail(ctx, DECXB_ERR_BAD_PARAM, std::string(name) + ": not aligned to its elements");
    if (ld < cols) return decxb_fail(ctx, DECXB_ERR_DIM_MISMATCH, std::string(name) + ": leading dimension smaller than the row length");
    return DECXB_OK;
}

/* Whether scratch may be taken on stream `s`: under capture it would outlive the call that owns it. */
inline int refuse_capture(decxb_ctx* ctx, cudaStream_t s, const char* what)
{
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    const cudaError_t e = cudaStreamIsCapturing(s, &st);
    if (e != cudaSuccess) cudaGetLastError();
    if (e != cudaSuccess || st != cudaStreamCaptureStatusNone)
        return decxb_fail(ctx, DECXB_ERR_BAD_PARAM, std::string("the stream is being captured and ") + what);
    return DECXB_OK;
}

/* Of the next launch; it alone leaves out the copies that decxb_inject_lost_copy names. */
inline Waits waits_of(decxb_ctx* ctx)
{
    const int64_t lost = ctx->lost_copy.load(std::memory_order_relaxed) < 0 ? -1 : ctx->lost_copy.exchange(-1);
    return {ctx->d_status, ctx->wait_limit_ns, (uint32_t)(ctx->wait_launches++ % 0xffffffffu) + 1u, lost};
}

}  // namespace fp8
#endif
