// Root-mean-square norm with the residual's addition:
//     s = x + r,   y = s / sqrt(mean(s^2) + eps) * w
// forward with y in the input's type, or as e4m3 codes with one E8M0 scale per 32 (the operand format of the block-scaled tensor-core
// GEMMs, the scale rule of dsv41/quant.py:46-54), and backward.  s leaves in the input's type (it is the residual of the next block); the
// norm itself uses the unrounded fp32 sum, and the backward pass adds x and r again instead of reading the rounded s, so that the only
// roundings are those of the outputs.
//
// All three are bound by HBM: a row is read once, held in registers (wide rows and most backward passes: in shared memory) and written once (forward 4
// arrays, 8-bit form 3.5, backward 5).
// A row belongs to tpr threads, each with NV vectors of 8 values (or single values where the width or an address does not allow 16-byte
// accesses); one reduction per row.  Measured (graph replay): bf16 one row of 4096 2.0 us; 8191 x 4096 46.5 us (5.8 TB/s); 4099 x 5120 in 8 bits
// 27.9 us (5.3 TB/s); 4099 x 16384 104 us (5.2 TB/s); fp32 8191 x 4096 83.5 us (6.4 TB/s); backward, the column sum of dw included, 8191 x 4096 61.9 us in
// bf16 (5.4 TB/s) and 131 in fp32 (5.1 TB/s).  Far from that: the backward pass of widths above 8192 (2048 x 16384 204 us in bf16, 1.6 TB/s) and of widths
// that are no multiple of 8 (8191 x 4095 252 us, 8191 x 4097 1535 us), whose register kernels spill 0.9 to 2.7 KB per thread above 8192 and, in single
// values, above 4096.
#include <cuda_fp8.h>

#include "b200_moe.h"
#include "common.cuh"
#include "dense.cuh"
#include "ftypes.cuh"
#include "tc5.cuh"

namespace b200 {

constexpr int NORM_MAX_DIM = 16384;
constexpr int NORM_MAX_STAGES = 8;
constexpr int NORM_RING_BYTES = 208 * 1024;  // of an SM, for the rings of its blocks

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

// Sum of NS values over the tpr threads of a row; every thread gets the totals.  Fixed order: within warps, then over the warps.  `red` (NS * 32 floats)
// must not be written again before every thread has passed another barrier: callers that walk rows alternate between two of them.
template <int NS>
__device__ __forceinline__ void row_sum(float (&v)[NS], int tpr, float* red) {
#pragma unroll
    for (int i = 0; i < NS; ++i) v[i] = warp_sum(v[i]);
    if (tpr == 32) return;
    const int nw = tpr >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;  // a row of more than 32 threads owns its block
    if (lane == 0)
#pragma unroll
        for (int i = 0; i < NS; ++i) red[i * 32 + warp] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NS; ++i) v[i] = warp_sum(lane < nw ? red[i * 32 + lane] : 0.f);
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

// y = s rinv w, stored as the call wants it
template <typename T, int VEC, int NV, bool QUANT, typename Weight>
__device__ __forceinline__ void norm_store(const NormArgs& a, long long row, bool live, int t, int tpr, float rinv, const float (&s)[NV][VEC], Weight weight) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (t + j * tpr) * VEC;
        const bool on = live && c < a.dim;
        float y[VEC];
        if (on) {
            float w[VEC];
            weight(j, c, w);
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
    norm_store<T, VEC, NV, QUANT>(a, row, live, t, tpr, rinv, s, [&](int, int c, float (&w)[VEC]) { load_weight<T, VEC>(a, c, w); });
}

// Many rows: the rows come by bulk copies into a ring of shared memory, which keeps the memory busy whatever the threads of a block wait for (16-byte
// aligned rows whose ring has three stages at least).  A row costs one barrier; once everybody has passed it the row's stage is refilled.
__device__ int g_norm_error = 0;
template <typename T, int NV, bool QUANT>
__global__ void __launch_bounds__(512) add_rms_norm_ring_kernel(const NormArgs a, int tpr, int stages) {
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ __align__(8) unsigned long long bars[NORM_MAX_STAGES];
    __shared__ float red[2][32];
    __shared__ int abort_flag;
    const int t = threadIdx.x;
    const uint32_t row_bytes = a.dim * (uint32_t)sizeof(T), stage_bytes = a.r ? 2 * row_bytes : row_bytes;
    if (t == 0) {
        abort_flag = 0;
        for (int i = 0; i < stages; ++i) mbar_init(smem_u32(&bars[i]), 1);
        mbar_fence_init();
    }
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();
    auto fetch = [&](long long row, int st) {  // one thread
        const uint32_t bar = smem_u32(&bars[st]), dst = smem_u32(ring) + st * stage_bytes;
        mbar_expect_tx(bar, stage_bytes);
        bulk_load(dst, reinterpret_cast<const T*>(a.x) + row * a.x_ld, row_bytes, bar);
        if (a.r) bulk_load(dst + row_bytes, reinterpret_cast<const T*>(a.r) + row * a.r_ld, row_bytes, bar);
    };
    if (t == 0)
        for (int i = 0; i < stages; ++i) {
            const long long row = blockIdx.x + (long long)i * gridDim.x;
            if (row < a.rows) fetch(row, i);
        }
    float w[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j)
        if ((t + j * tpr) * 8 < a.dim) load_weight<T, 8>(a, (t + j * tpr) * 8, w[j]);
    int st = 0, turn = 0;
    uint32_t ph = 0;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        mbar_wait(smem_u32(&bars[st]), ph, &abort_flag, &g_norm_error, 2);  // a wait that gives up leaves wrong rows, not a hang
        const T* x = reinterpret_cast<const T*>(ring + st * stage_bytes);
        float s[NV][8], ss[1] = {0.f};
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (t + j * tpr) * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) s[j][i] = 0.f;
            if (c < a.dim) {
                load8<T>(x + c, s[j]);
                if (a.r) {
                    float v[8];
                    load8<T>(x + a.dim + c, v);
#pragma unroll
                    for (int i = 0; i < 8; ++i) s[j][i] += v[i];
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) ss[0] += s[j][i] * s[j][i];
            }
        }
        if (tpr == 32) __syncwarp();
        row_sum<1>(ss, tpr, red[turn]);
        turn ^= 1;
        const long long ahead = row + (long long)stages * gridDim.x;
        if (t == 0 && ahead < a.rows) fetch(ahead, st);
        if (++st == stages) { st = 0; ph ^= 1; }
        const float rinv = rsqrtf(ss[0] / (float)a.dim + a.eps);
        norm_store<T, 8, NV, QUANT>(a, row, true, t, tpr, rinv, s, [&](int j, int, float (&v)[8]) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = w[j][i];
        });
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
    __shared__ float red[2][64];
    pdl_wait();
    pdl_launch_dependents();
    const int t = threadIdx.x;  // one row per block pass: blockDim.x == tpr
    int turn = 0;
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
        row_sum<2>(sum, tpr, red[turn]);
        turn ^= 1;
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

// The same with the rows fetched by bulk copies into a ring of shared memory, as in the forward pass.
template <typename T, int NV>
__global__ void __launch_bounds__(512) add_rms_norm_bwd_ring_kernel(const NormArgs a, int tpr, int stages) {
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ __align__(8) unsigned long long bars[NORM_MAX_STAGES];
    __shared__ float red[2][64];
    __shared__ int abort_flag;
    const int t = threadIdx.x;
    const uint32_t row_bytes = a.dim * (uint32_t)sizeof(T), arrays = 2 + (a.r != nullptr) + (a.gs != nullptr), stage_bytes = arrays * row_bytes;
    if (t == 0) {
        abort_flag = 0;
        for (int i = 0; i < stages; ++i) mbar_init(smem_u32(&bars[i]), 1);
        mbar_fence_init();
    }
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();
    auto fetch = [&](long long row, int st) {  // one thread
        const uint32_t bar = smem_u32(&bars[st]);
        uint32_t dst = smem_u32(ring) + st * stage_bytes;
        mbar_expect_tx(bar, stage_bytes);
        bulk_load(dst, reinterpret_cast<const T*>(a.x) + row * a.x_ld, row_bytes, bar);
        bulk_load(dst += row_bytes, reinterpret_cast<const T*>(a.gy) + row * a.dim, row_bytes, bar);
        if (a.r) bulk_load(dst += row_bytes, reinterpret_cast<const T*>(a.r) + row * a.r_ld, row_bytes, bar);
        if (a.gs) bulk_load(dst += row_bytes, reinterpret_cast<const T*>(a.gs) + row * a.dim, row_bytes, bar);
    };
    if (t == 0)
        for (int i = 0; i < stages; ++i) {
            const long long row = blockIdx.x + (long long)i * gridDim.x;
            if (row < a.rows) fetch(row, i);
        }
    float dw[NV][8], w[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[j][i] = w[j][i] = 0.f;
        if ((t + j * tpr) * 8 < a.dim) load_weight<T, 8>(a, (t + j * tpr) * 8, w[j]);
    }
    int st = 0, turn = 0;
    uint32_t ph = 0;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        mbar_wait(smem_u32(&bars[st]), ph, &abort_flag, &g_norm_error, 1);  // a wait that gives up leaves wrong sums, not a hang
        const T* x = reinterpret_cast<const T*>(ring + st * stage_bytes);
        const T *gy = x + a.dim, *r = gy + a.dim, *gs = a.r ? r + a.dim : r;
        float s[NV][8], g[NV][8], d[NV][8];
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (t + j * tpr) * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) s[j][i] = g[j][i] = d[j][i] = 0.f;
            if (c < a.dim) {
                load8<T>(x + c, s[j]);
                load8<T>(gy + c, g[j]);
                if (a.r) {
                    float v[8];
                    load8<T>(r + c, v);
#pragma unroll
                    for (int i = 0; i < 8; ++i) s[j][i] += v[i];
                }
                if (a.gs) load8<T>(gs + c, d[j]);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    sum[0] += s[j][i] * s[j][i];
                    sum[1] += g[j][i] * w[j][i] * s[j][i];
                }
            }
        }
        if (tpr == 32) __syncwarp();
        row_sum<2>(sum, tpr, red[turn]);
        turn ^= 1;
        const long long ahead = row + (long long)stages * gridDim.x;
        if (t == 0 && ahead < a.rows) fetch(ahead, st);
        if (++st == stages) { st = 0; ph ^= 1; }
        const float rinv = rsqrtf(sum[0] / (float)a.dim + a.eps);
        const float k = rinv * rinv * (sum[1] / (float)a.dim);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (t + j * tpr) * 8;
            if (c < a.dim) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    d[j][i] += rinv * (g[j][i] * w[j][i] - s[j][i] * k);
                    dw[j][i] += g[j][i] * (s[j][i] * rinv);
                }
                store8<T>(reinterpret_cast<T*>(a.ds) + row * a.dim + c, d[j]);
            }
        }
    }
    if (a.dw_part) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (t + j * tpr) * 8;
            if (c < a.dim) store8<float>(a.dw_part + (long long)blockIdx.x * a.dim + c, dw[j]);
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

template <typename T, int NV, bool QUANT>
static int fwd_ring(const NormArgs& a, int tpr, int stages, size_t smem, int grid, cudaStream_t stream) {
    auto kernel = add_rms_norm_ring_kernel<T, NV, QUANT>;
    static bool attr_done[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !attr_done[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, NORM_RING_BYTES);
        if (e != cudaSuccess) return (int)e;
        if (dev >= 0 && dev < 64) attr_done[dev] = true;
    }
    return (int)launch_pdl(kernel, dim3(grid), dim3(tpr), smem, stream, a, tpr, stages);
}

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
        // Many rows of more than 8 KB: the ring (4099 x 5120 in 8 bits 27.9 us against 32.2, 2000 x 8192 22.7 against 28.5); shorter rows take more time
        // per barrier than they give the memory to do (8191 x 4096: 49.5 against 46.2).
        const int rtpr = threads_per_row(a.dim, 8, 2);
        if (a.rows > 2 * sm_count() && a.dim * sizeof(T) > 8192 && rtpr <= 512) {
            const int per_sm = 1024 / rtpr;
            const size_t stage = (size_t)(a.r ? 2 : 1) * a.dim * sizeof(T);
            int stages = (int)(NORM_RING_BYTES / per_sm / stage);
            if (stages > NORM_MAX_STAGES) stages = NORM_MAX_STAGES;
            const long long cap = (long long)sm_count() * per_sm;
            if (stages >= 3) return fwd_ring<T, 2, QUANT>(a, rtpr, stages, stages * stage, (int)(a.rows < cap ? a.rows : cap), stream);
        }
        // Few rows: as many threads as there are vectors (64 x 4096: 2.4 us with one vector per thread, 2.8 with two, 4.1 with four).  Many rows:
        // blocks of about 300 threads, several per SM, so that some load while others reduce (8191 x 4096: 46.6 us against 54.8 with one vector per
        // thread).
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
    int nv = vec ? 2 : (dim <= 1024 * 4 ? 4 : 16);
    while (vec && threads_per_row(dim, 8, nv) > 512) nv *= 2;
    return {nv, threads_per_row(dim, vec ? 8 : 1, nv)};
}

// blocks per SM of the backward pass
static int norm_bwd_per_sm(int dim) {
    const int n = 512 / norm_bwd_shape(dim, true).tpr;
    return n > 16 ? 16 : n;
}

template <typename T>
static int bwd_ring(const NormArgs& a, int tpr, int stages, size_t smem, int grid, cudaStream_t stream) {
    auto kernel = add_rms_norm_bwd_ring_kernel<T, 2>;
    static bool attr_done[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !attr_done[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, NORM_RING_BYTES);
        if (e != cudaSuccess) return (int)e;
        if (dev >= 0 && dev < 64) attr_done[dev] = true;
    }
    return (int)launch_pdl(kernel, dim3(grid), dim3(tpr), smem, stream, a, tpr, stages);
}

template <typename T>
static int bwd_typed(const NormArgs& a, bool vec, int grid, cudaStream_t stream) {
    const BwdShape b = norm_bwd_shape(a.dim, vec);
    if (vec && b.nv == 2) {
        const size_t stage = (size_t)(2 + (a.r != nullptr) + (a.gs != nullptr)) * a.dim * sizeof(T);
        int stages = (int)(NORM_RING_BYTES / norm_bwd_per_sm(a.dim) / stage);
        if (stages > NORM_MAX_STAGES) stages = NORM_MAX_STAGES;
        if (stages >= 3) return bwd_ring<T>(a, b.tpr, stages, stages * stage, grid, stream);
    }
    void (*k)(const NormArgs, int) = vec ? (b.nv == 2 ? add_rms_norm_bwd_kernel<T, 8, 2> : add_rms_norm_bwd_kernel<T, 8, 4>)
                                         : (b.nv == 4 ? add_rms_norm_bwd_kernel<T, 1, 4> : add_rms_norm_bwd_kernel<T, 1, 16>);
    return (int)launch_pdl(k, dim3(grid), dim3(b.tpr), 0, stream, a, b.tpr);
}

// about 512 threads per SM walk the rows (8191 x 4096: 60.9 us with two blocks of 256 per SM, 79.6 with one of 512, 72.1 with one of 256); the same for both vector widths, so that the workspace does not depend on the addresses
static int norm_bwd_grid(long long rows, int dim) {
    const long long cap = (long long)sm_count() * norm_bwd_per_sm(dim);
    return (int)(rows < cap ? rows : cap);
}

int norm_device_error(int* out) {
    int v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, g_norm_error, sizeof(int));
    if (e != cudaSuccess) return (int)e;
    if (v) {
        int z = 0;
        cudaMemcpyToSymbol(g_norm_error, &z, sizeof(int));
    }
    *out = v;
    return 0;
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
