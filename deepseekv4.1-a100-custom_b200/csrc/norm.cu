// Root-mean-square norm with the residual's addition:
//     s = x + r,   y = s / sqrt(mean(s^2) + eps) * w
// forward with y in the input's type, or as e4m3 codes with one E8M0 scale per 32 (the operand format of the block-scaled tensor-core
// GEMMs, the scale rule of dsv41/quant.py:46-54), and backward.  s leaves in the input's type (it is the residual of the next block); the
// norm itself uses the unrounded fp32 sum, and the backward pass adds x and r again instead of reading the rounded s, so that the only
// roundings are those of the outputs.
//
// All three are bound by HBM: a row is read once, held in registers as fp32 and written once (forward 4 arrays, 8-bit form 3.03, backward 5).
// A row belongs to TPR threads, each with NV vectors of 8 values (or single values where the width or an address does not allow 16-byte
// accesses); one reduction per row.
#include <cuda_fp8.h>

#include "b200_moe.h"
#include "common.cuh"
#include "dense.cuh"
#include "ftypes.cuh"

namespace b200 {

constexpr int NORM_MAX_DIM = 16384;

struct NormArgs {
    const void *x, *r, *w;
    long long x_ld, r_ld;
    int w_f32;
    long long rows;
    int dim;
    float eps;
    void *y, *s;
    uint8_t *q8, *sf;
    // backward
    const void *gy, *gs;
    void* ds;
    float* dw_part;  // [gridDim.x][dim]
};

// Sum of NS values over the TPR threads of a row; every thread gets the totals.  Fixed order.
template <int NS>
__device__ __forceinline__ void row_sum(float (&v)[NS], int tpr, float* red) {
#pragma unroll
    for (int i = 0; i < NS; ++i) v[i] = warp_sum(v[i]);
    if (tpr == 32) return;
    const int nw = tpr >> 5, warp = threadIdx.x >> 5;  // a row of more than 32 threads owns its block
    __syncthreads();                                   // the totals of the row before have been read
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int i = 0; i < NS; ++i) red[i * 32 + warp] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        float t = 0.f;
        for (int k = 0; k < nw; ++k) t += red[i * 32 + k];
        v[i] = t;
    }
}

template <typename T, int VEC>
__device__ __forceinline__ void load_weight(const NormArgs& a, int c, float (&w)[VEC]) {
    if (!a.w) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) w[i] = 1.f;
    } else if (a.w_f32) {
        load_vec<float, VEC>(reinterpret_cast<const float*>(a.w) + c, w);
    } else {
        load_vec<T, VEC>(reinterpret_cast<const T*>(a.w) + c, w);
    }
}

template <typename T, int VEC, int NV, bool QUANT>
__global__ void __launch_bounds__(1024) add_rms_norm_kernel(const NormArgs a, int tpr) {
    __shared__ float red[32];
    pdl_wait();
    pdl_launch_dependents();
    const int t = tpr == 32 ? threadIdx.x & 31 : threadIdx.x;  // several rows of 32 threads per block, or one of more
    const long long row = tpr == 32 ? (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    const bool live = row < a.rows;  // a dead row's threads still take part in the shuffles
    const T* x = reinterpret_cast<const T*>(a.x) + (live ? row : 0) * a.x_ld;
    const T* r = a.r ? reinterpret_cast<const T*>(a.r) + (live ? row : 0) * a.r_ld : nullptr;
    float s[NV][VEC];
    float ss[1] = {0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (t + j * tpr) * VEC;
        const bool on = live && c < a.dim;
#pragma unroll
        for (int i = 0; i < VEC; ++i) s[j][i] = 0.f;
        if (on) {
            load_vec<T, VEC>(x + c, s[j]);
            if (r) {
                float v[VEC];
                load_vec<T, VEC>(r + c, v);
#pragma unroll
                for (int i = 0; i < VEC; ++i) s[j][i] += v[i];
            }
        }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) ss[0] += s[j][i] * s[j][i];
    row_sum<1>(ss, tpr, red);
    const float rinv = rsqrtf(ss[0] / (float)a.dim + a.eps);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (t + j * tpr) * VEC;
        const bool on = live && c < a.dim;
        float y[VEC];
        if (on) {
            float w[VEC];
            load_weight<T, VEC>(a, c, w);
            if (a.s) store_vec<T, VEC>(reinterpret_cast<T*>(a.s) + row * a.dim + c, s[j]);
#pragma unroll
            for (int i = 0; i < VEC; ++i) y[i] = s[j][i] * rinv * w[i];
            if (a.y) store_vec<T, VEC>(reinterpret_cast<T*>(a.y) + row * a.dim + c, y);
        }
        if constexpr (QUANT) {
            float amax = 0.f;
            if (on)
#pragma unroll
                for (int i = 0; i < VEC; ++i) amax = fmaxf(amax, fabsf(y[i]));
            // a group of 32 = 4 threads with 8 values or one warp (dim % 32 == 0: its threads are on or off together)
#pragma unroll
            for (int o = VEC == 8 ? 2 : 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            if (!on) continue;
            // ceil(log2(amax / 448)) from the bits: amax = M 2^E, 448 = 1.75 * 2^8.  An infinite amax takes the largest finite scale.
            const uint32_t b = f32_as_u32(fminf(fmaxf(amax, 1e-4f), 3.3e38f));
            const uint32_t sb = (b >> 23) - 8 + ((b & 0x7FFFFF) > 0x600000 ? 1 : 0);
            const float inv = u32_as_f32((254u - sb) << 23);  // 1 / scale, exact
            uint8_t* q = a.q8 + row * a.dim + c;
            if constexpr (VEC == 8) {
                uint32_t o[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[4 * h] * inv, y[4 * h + 1] * inv), __NV_SATFINITE, __NV_E4M3);
                    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[4 * h + 2] * inv, y[4 * h + 3] * inv), __NV_SATFINITE, __NV_E4M3);
                    o[h] = lo | (hi << 16);
                }
                *reinterpret_cast<uint2*>(q) = make_uint2(o[0], o[1]);
            } else {
                *q = (uint8_t)__nv_cvt_float_to_fp8(y[0] * inv, __NV_SATFINITE, __NV_E4M3);
            }
            if ((c & 31) == 0) a.sf[row * (a.dim >> 5) + (c >> 5)] = (uint8_t)sb;
        }
    }
}

// Backward.  With n = s rinv and h = gy w:  ds = rinv (h - n mean(h n)) + gs,  dw = sum over rows of gy n.
// Blocks walk the rows with the grid's stride and keep their part of dw in registers; the parts are added in block order by
// column_sum_kernel (no atomics: the same result from run to run).  The next row's loads are issued before this row's reduction, so that the
// memory works through the barriers.
template <typename T, int VEC> struct RawVec { static constexpr int WORDS = sizeof(T) * VEC / 4; uint32_t u[WORDS]; };
template <typename T> struct RawVec<T, 1> { T u; };

template <typename T, int VEC>
__device__ __forceinline__ void load_raw(const T* p, RawVec<T, VEC>& r) {
    if constexpr (VEC == 1) r.u = *p;
    else
#pragma unroll
        for (int i = 0; i < RawVec<T, VEC>::WORDS / 4; ++i) {
            const uint4 q = reinterpret_cast<const uint4*>(p)[i];
            r.u[4 * i] = q.x; r.u[4 * i + 1] = q.y; r.u[4 * i + 2] = q.z; r.u[4 * i + 3] = q.w;
        }
}
template <typename T, int VEC>
__device__ __forceinline__ void value_of(const RawVec<T, VEC>& r, float (&v)[VEC]) {
    if constexpr (VEC == 1) v[0] = to_f32(r.u);
    else if constexpr (sizeof(T) == 4)
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = __uint_as_float(r.u[i]);
    else
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
            const float2 f = unpack2<T>(r.u[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
}

template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(VEC == 8 ? 512 : 1024) add_rms_norm_bwd_kernel(const NormArgs a, int tpr) {
    __shared__ float red[64];
    pdl_wait();
    pdl_launch_dependents();
    const int t = threadIdx.x;  // one row per block pass: blockDim.x == tpr
    float dw[NV][VEC];
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) dw[j][i] = 0.f;
    RawVec<T, VEC> rx[NV], rr[NV], rg[NV], rs[NV];
    auto fetch = [&](long long row) {
        const T* x = reinterpret_cast<const T*>(a.x) + row * a.x_ld;
        const T* r = a.r ? reinterpret_cast<const T*>(a.r) + row * a.r_ld : nullptr;
        const T* gy = reinterpret_cast<const T*>(a.gy) + row * a.dim;
        const T* gs = a.gs ? reinterpret_cast<const T*>(a.gs) + row * a.dim : nullptr;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (t + j * tpr) * VEC;
            if (c < a.dim) {
                load_raw<T, VEC>(x + c, rx[j]);
                load_raw<T, VEC>(gy + c, rg[j]);
                if (r) load_raw<T, VEC>(r + c, rr[j]);
                if (gs) load_raw<T, VEC>(gs + c, rs[j]);
            }
        }
    };
    if (blockIdx.x < a.rows) fetch(blockIdx.x);
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        float s[NV][VEC], g[NV][VEC], d[NV][VEC];
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (t + j * tpr) * VEC;
#pragma unroll
            for (int i = 0; i < VEC; ++i) s[j][i] = g[j][i] = d[j][i] = 0.f;
            if (c < a.dim) {
                float w[VEC], v[VEC];
                load_weight<T, VEC>(a, c, w);
                value_of<T, VEC>(rx[j], s[j]);
                value_of<T, VEC>(rg[j], g[j]);
                if (a.r) {
                    value_of<T, VEC>(rr[j], v);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) s[j][i] += v[i];
                }
                if (a.gs) value_of<T, VEC>(rs[j], d[j]);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    sum[0] += s[j][i] * s[j][i];
                    sum[1] += g[j][i] * w[i] * s[j][i];
                }
            }
        }
        if (row + gridDim.x < a.rows) fetch(row + gridDim.x);
        row_sum<2>(sum, tpr, red);
        const float rinv = rsqrtf(sum[0] / (float)a.dim + a.eps);
        const float k = rinv * rinv * (sum[1] / (float)a.dim);  // n mean(h n) = s rinv * rinv mean(h s)
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (t + j * tpr) * VEC;
            if (c < a.dim) {
                float w[VEC];
                load_weight<T, VEC>(a, c, w);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    d[j][i] += rinv * (g[j][i] * w[i] - s[j][i] * k);
                    dw[j][i] += g[j][i] * (s[j][i] * rinv);
                }
                store_vec<T, VEC>(reinterpret_cast<T*>(a.ds) + row * a.dim + c, d[j]);
            }
        }
    }
    if (a.dw_part) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (t + j * tpr) * VEC;
            if (c < a.dim) store_vec<float, VEC>(a.dw_part + (long long)blockIdx.x * a.dim + c, dw[j]);
        }
    }
}

// out[c] = sum of part[p][c] over p, in a fixed order: 32 slices of the parts by the 32 warps of a block, then the slices
template <typename T>
__global__ void __launch_bounds__(1024) column_sum_kernel(const float* __restrict__ part, int parts, int dim, T* __restrict__ out) {
    __shared__ float red[32][33];
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, sl = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float acc = 0.f;
    if (c < dim) {
#pragma unroll 8
        for (int p = sl; p < parts; p += 32) acc += part[(long long)p * dim + c];
    }
    red[sl][lane] = acc;
    __syncthreads();
    if (sl == 0 && c < dim) {
#pragma unroll
        for (int i = 1; i < 32; ++i) acc += red[i][lane];
        out[c] = from_f32<T>(acc);
    }
}

int column_sum(const float* part, int parts, int dim, int dtype, void* out, cudaStream_t stream) {
    const dim3 g((dim + 31) / 32), b(1024);
    if (dtype == F_FP32) return (int)launch_pdl(column_sum_kernel<float>, g, b, 0, stream, part, parts, dim, (float*)out);
    if (dtype == F_BF16) return (int)launch_pdl(column_sum_kernel<__nv_bfloat16>, g, b, 0, stream, part, parts, dim, (__nv_bfloat16*)out);
    return (int)launch_pdl(column_sum_kernel<__half>, g, b, 0, stream, part, parts, dim, (__half*)out);
}

// ------------------------------------------------------------------ host
int sm_count();

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// threads per row, whole warps, so that a thread holds at most `nv` vectors
static int threads_per_row(int dim, int vec, int nv) { return (dim + vec * nv * 32 - 1) / (vec * nv * 32) * 32; }

template <typename T, int VEC, int NV, bool QUANT>
static int launch_fwd(const NormArgs& a, int tpr, cudaStream_t stream) {
    const int rpb = tpr == 32 ? 4 : 1;
    const long long grid = (a.rows + rpb - 1) / rpb;
    if (grid > 0x7FFFFFFFll) return ERR_TOO_LARGE;
    return (int)launch_pdl(add_rms_norm_kernel<T, VEC, NV, QUANT>, dim3((unsigned)grid), dim3(tpr * rpb), 0, stream, a, tpr);
}

template <typename T, bool QUANT>
static int fwd_typed(const NormArgs& a, bool vec, cudaStream_t stream) {
    if (vec) {
        // Few rows: as many threads as there are vectors (64 x 4096: 2.4 us with one vector per thread, 2.8 with two, 4.1 with four).  Many rows:
        // blocks of about 300 threads, several per SM, so that some load while others reduce (4099 x 5120: 32.6 us against 38.2 with one
        // vector per thread; 2000 x 8192: 28.8 with four against 33.0).
        int nv = 1;
        while (threads_per_row(a.dim, 8, nv) > (a.rows <= sm_count() ? 1024 : 320) && nv < 4) nv *= 2;
        if (nv == 1) return launch_fwd<T, 8, 1, QUANT>(a, threads_per_row(a.dim, 8, 1), stream);
        if (nv == 2) return launch_fwd<T, 8, 2, QUANT>(a, threads_per_row(a.dim, 8, 2), stream);
        return launch_fwd<T, 8, 4, QUANT>(a, threads_per_row(a.dim, 8, 4), stream);
    }
    if (a.dim <= 1024 * 4) return launch_fwd<T, 1, 4, QUANT>(a, threads_per_row(a.dim, 1, 4), stream);
    return launch_fwd<T, 1, 16, QUANT>(a, threads_per_row(a.dim, 1, 16), stream);
}

// threads of a row and vectors a thread holds in the backward pass (dim <= NORM_MAX_DIM: at most 512 threads of 4 vectors)
struct BwdShape { int nv, tpr; };
static BwdShape norm_bwd_shape(int dim, bool vec) {
    int nv = vec ? 1 : (dim <= 1024 * 4 ? 4 : 16);
    while (vec && threads_per_row(dim, 8, nv) > 512) nv *= 2;
    return {nv, threads_per_row(dim, vec ? 8 : 1, nv)};
}

template <typename T>
static int bwd_typed(const NormArgs& a, bool vec, int grid, cudaStream_t stream) {
    const BwdShape b = norm_bwd_shape(a.dim, vec);
    void (*k)(const NormArgs, int) = vec ? (b.nv == 1 ? add_rms_norm_bwd_kernel<T, 8, 1> : b.nv == 2 ? add_rms_norm_bwd_kernel<T, 8, 2> : add_rms_norm_bwd_kernel<T, 8, 4>)
                                         : (b.nv == 4 ? add_rms_norm_bwd_kernel<T, 1, 4> : add_rms_norm_bwd_kernel<T, 1, 16>);
    return (int)launch_pdl(k, dim3(grid), dim3(b.tpr), 0, stream, a, b.tpr);
}

// about 512 threads per SM walk the rows (8191 x 4096: 82.5 us with one block of 512 per SM, 87.8 with four; 4096 x 1024: 15.6 with four of 128);
// the same for both vector widths, so that the workspace does not depend on the addresses
static int norm_bwd_grid(long long rows, int dim) {
    int per_sm = 512 / norm_bwd_shape(dim, true).tpr;
    if (per_sm > 16) per_sm = 16;
    const long long cap = (long long)sm_count() * per_sm;
    return (int)(rows < cap ? rows : cap);
}

}  // namespace b200

using namespace b200;

static int norm_check(const void* x, long long x_ld, const void* r, long long r_ld, int dtype, long long rows, int dim, float eps) {
    if (rows < 0 || dim <= 0 || !(eps >= 0.f)) return ERR_BAD_ARG;
    if (dtype < F_BF16 || dtype > F_FP32) return ERR_UNSUPPORTED;
    if (dim > NORM_MAX_DIM) return ERR_TOO_LARGE;
    if (rows > 0 && !x) return ERR_BAD_ARG;
    if (rows > 1 && ((x_ld < dim) || (r && r_ld < dim))) return ERR_BAD_SHAPE;
    return 0;
}

extern "C" int b200_add_rms_norm(const void* x, long long x_ld, const void* residual, long long r_ld, const void* w, int w_is_f32, int dtype, long long rows,
                                 int dim, float eps, void* y, void* sum, void* q8, void* sf, cudaStream_t stream) {
    const int rc = norm_check(x, x_ld, residual, r_ld, dtype, rows, dim, eps);
    if (rc) return rc;
    if (q8 && dim % 32) return ERR_BAD_SHAPE;
    if (rows == 0) return 0;
    if ((!y && !q8) || (q8 && !sf)) return ERR_BAD_ARG;
    NormArgs a{};
    a.x = x; a.r = residual; a.w = w; a.x_ld = x_ld; a.r_ld = r_ld; a.w_f32 = w_is_f32; a.rows = rows; a.dim = dim; a.eps = eps;
    a.y = y; a.s = sum; a.q8 = (uint8_t*)q8; a.sf = (uint8_t*)sf;
    const int per16 = 16 / f_elem_bytes(dtype);
    const bool vec = dim % 8 == 0 && aligned16(x) && aligned16(residual) && aligned16(w) && aligned16(y) && aligned16(sum) && ((uintptr_t)q8 & 7) == 0 &&
                     x_ld % per16 == 0 && (!residual || r_ld % per16 == 0);
    if (dtype == F_BF16) return q8 ? fwd_typed<__nv_bfloat16, true>(a, vec, stream) : fwd_typed<__nv_bfloat16, false>(a, vec, stream);
    if (dtype == F_FP16) return q8 ? fwd_typed<__half, true>(a, vec, stream) : fwd_typed<__half, false>(a, vec, stream);
    return q8 ? fwd_typed<float, true>(a, vec, stream) : fwd_typed<float, false>(a, vec, stream);
}

extern "C" size_t b200_add_rms_norm_bwd_workspace_bytes(long long rows, int dim) {
    if (rows <= 0 || dim <= 0) return 0;
    return (size_t)norm_bwd_grid(rows, dim) * (size_t)dim * sizeof(float);
}

extern "C" int b200_add_rms_norm_bwd(const void* x, long long x_ld, const void* residual, long long r_ld, const void* w, int w_is_f32, int dtype, long long rows,
                                     int dim, float eps, const void* gy, const void* gsum, void* ds, void* dw, void* workspace, size_t workspace_bytes,
                                     cudaStream_t stream) {
    const int rc = norm_check(x, x_ld, residual, r_ld, dtype, rows, dim, eps);
    if (rc) return rc;
    if (rows > 0 && (!gy || !ds)) return ERR_BAD_ARG;
    if (dw && !w) return ERR_BAD_ARG;
    if (rows == 0) return dw ? (int)cudaMemsetAsync(dw, 0, (size_t)dim * (w_is_f32 ? 4 : f_elem_bytes(dtype)), stream) : 0;
    if (dw && (!workspace || workspace_bytes < b200_add_rms_norm_bwd_workspace_bytes(rows, dim))) return ERR_WORKSPACE;
    if (dw && !aligned16(workspace)) return ERR_BAD_ALIGN;
    const int grid = norm_bwd_grid(rows, dim);
    NormArgs a{};
    a.x = x; a.r = residual; a.w = w; a.x_ld = x_ld; a.r_ld = r_ld; a.w_f32 = w_is_f32; a.rows = rows; a.dim = dim; a.eps = eps;
    a.gy = gy; a.gs = gsum; a.ds = ds; a.dw_part = dw ? (float*)workspace : nullptr;
    const int per16 = 16 / f_elem_bytes(dtype);
    const bool vec = dim % 8 == 0 && aligned16(x) && aligned16(residual) && aligned16(w) && aligned16(gy) && aligned16(gsum) && aligned16(ds) && x_ld % per16 == 0 &&
                     (!residual || r_ld % per16 == 0);
    int e = dtype == F_BF16 ? bwd_typed<__nv_bfloat16>(a, vec, grid, stream)
            : dtype == F_FP16 ? bwd_typed<__half>(a, vec, grid, stream) : bwd_typed<float>(a, vec, grid, stream);
    if (e || !dw) return e;
    return column_sum((const float*)workspace, grid, dim, w_is_f32 ? (int)F_FP32 : dtype, dw, stream);
}
