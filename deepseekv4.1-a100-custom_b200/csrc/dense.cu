// C entry points of the dense feed-forward operators: out = act(x W^T + bias) + residual and the gated product
// act(x Wg^T) * (x Wu^T), with the element-wise halves of their backward passes.  The products are fgemm.cu's.
#include "b200_moe.h"
#include "common.cuh"
#include "dense.cuh"
#include "fgemm.cuh"
#include "ftypes.cuh"

namespace b200 {

// dz = gy * act'(z) and the column sums of dz.  z arrives in fp32: in 16 bits its rounding would put an error of the size of the result's own
// rounding into every gradient.  dz leaves in T, since the tensor cores multiply 16-bit values (as torch's 16-bit linear does): the gradients' error against
// 64 bits is 0.00029 in place of 0.00021 of an fp32 dz in fp16, 0.0023 in place of 0.0017 in bf16.  8 warps of a block share DZ_ROWS rows of 32 * VEC columns; the sums of a block's rows go to
// part[row block][N] in fp32 (from the unrounded dz), added in block order afterwards.  Row and column blocks share grid x (y ends at 65535, which would
// end the rows at 4.2 million).  Bound by HBM: gy and z in, dz out.
constexpr int DZ_ROWS = 64;
template <typename T, int VEC>
__global__ void __launch_bounds__(256) act_bwd_kernel(const T* __restrict__ gy, long long gy_ld, const float* __restrict__ z, long long z_ld, int act, int M, int N,
                                                      T* __restrict__ dz, long long dz_ld, float* __restrict__ part, int col_blocks) {
    __shared__ float red[8][32 * VEC];
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rb = blockIdx.x / col_blocks, cb = blockIdx.x - rb * col_blocks;
    const int c = (cb * 32 + lane) * VEC;
    const int r_end = min(M, (rb + 1) * DZ_ROWS);
    float sum[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum[i] = 0.f;
    if (c < N) {
        for (int r = rb * DZ_ROWS + warp; r < r_end; r += 8) {
            float g[VEC];
            load_vec<T, VEC>(gy + r * gy_ld + c, g);
            if (z) {
                float v[VEC], y[VEC], d[VEC];
                load_vec<float, VEC>(z + r * z_ld + c, v);
                act_bwd_n(act, v, y, d);
#pragma unroll
                for (int i = 0; i < VEC; ++i) g[i] *= d[i];
            }
            if (dz) store_vec<T, VEC>(dz + r * dz_ld + c, g);
#pragma unroll
            for (int i = 0; i < VEC; ++i) sum[i] += g[i];
        }
    }
    if (!part) return;
#pragma unroll
    for (int i = 0; i < VEC; ++i) red[warp][i * 32 + lane] = sum[i];
    __syncthreads();
    for (int k = threadIdx.x; k < 32 * VEC; k += 256) {
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) t += red[w][k];
        const int col = (cb * 32 + (k & 31)) * VEC + (k >> 5);
        if (col < N) part[(long long)rb * N + col] = t;
    }
}

// [dg | du] of the gated product from gy and the saved [g | u]: dg = gy u' act'(g') where the clamp let g through, du = gy act(g') where it
// let u through (g', u': the clamped values).  g and u arrive in fp32, dg and du leave in T (as z and dz above).  Bound by HBM: 10 bytes in, 4 out per element of gy.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) gated_bwd_kernel(const T* __restrict__ gy, long long gy_ld, const float* __restrict__ gu, long long gu_ld, int act, float limit, long long M,
                                                        int inter, T* __restrict__ dgu, long long dgu_ld) {
    pdl_wait();
    pdl_launch_dependents();
    const int per_row = (inter + VEC - 1) / VEC;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long r = i <= 0xFFFFFFFFll ? (uint32_t)i / (uint32_t)per_row : i / per_row;  // a 64-bit division is 5 times the instructions
    if (r >= M) return;
    const int c = (int)(i - r * per_row) * VEC;
    float d[VEC], g[VEC], u[VEC];
    load_vec<T, VEC>(gy + r * gy_ld + c, d);
    load_vec<float, VEC>(gu + r * gu_ld + c, g);
    load_vec<float, VEC>(gu + r * gu_ld + inter + c, u);
    float pass_g[VEC], pass_u[VEC], a[VEC], da[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
        pass_g[k] = pass_u[k] = d[k];
        if (limit > 0.f) {
            if (g[k] > limit) { g[k] = limit; pass_g[k] = 0.f; }
            if (fabsf(u[k]) > limit) { u[k] = copysignf(limit, u[k]); pass_u[k] = 0.f; }
        }
    }
    act_bwd_n(act, g, a, da);
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
        g[k] = pass_g[k] * u[k] * da[k];
        u[k] = pass_u[k] * a[k];
    }
    store_vec<T, VEC>(dgu + r * dgu_ld + c, g);
    store_vec<T, VEC>(dgu + r * dgu_ld + inter + c, u);
}

// Rows of any width and address into rows that start on 16 bytes (dst_ld a multiple of 8): a tensor map needs that.  One or two matrices of
// the same width in a launch.
struct AlignRows { const uint16_t* src; long long src_ld; uint16_t* dst; long long rows; };
__global__ void __launch_bounds__(256) align_rows_kernel(const AlignRows m0, const AlignRows m1, long long dst_ld, int cols) {
    pdl_wait();
    pdl_launch_dependents();
    const int per_row = (cols + 7) / 8;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x, ri = i / per_row;
    if (ri >= m0.rows + m1.rows) return;
    const bool second = ri >= m0.rows;
    const long long r = second ? ri - m0.rows : ri;
    const int c = (int)(i - ri * per_row) * 8;
    const uint16_t* s = (second ? m1.src + r * m1.src_ld : m0.src + r * m0.src_ld) + c;
    uint32_t v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = c + k < cols ? s[k] : 0;  // the rest of the last 16 bytes: zeros
    *reinterpret_cast<uint4*>((second ? m1.dst : m0.dst) + r * dst_ld + c) = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
}

static bool ok16(const void* p, long long ld) { return !((uintptr_t)p & 15) && ld % 8 == 0; }  // rows start on 16 bytes (fp32: on 32)

template <typename T>
static int act_bwd_run(const void* gy, long long gy_ld, const float* z, long long z_ld, int act, int M, int N, void* dz, long long dz_ld, float* part, cudaStream_t stream) {
    const bool vec = N % 8 == 0 && ok16(gy, gy_ld) && (!z || ok16(z, z_ld)) && (!dz || ok16(dz, dz_ld));
    const int w = vec ? 256 : 32, col_blocks = (N + w - 1) / w;
    const long long blocks = (long long)((M + DZ_ROWS - 1) / DZ_ROWS) * col_blocks;
    if (blocks > 0x7FFFFFFFll) return ERR_TOO_LARGE;
    return (int)launch_pdl(vec ? act_bwd_kernel<T, 8> : act_bwd_kernel<T, 1>, dim3((unsigned)blocks), dim3(256), 0, stream, (const T*)gy, gy_ld, z, z_ld, act, M, N, (T*)dz,
                           dz_ld, part, col_blocks);
}

template <typename T>
static int gated_bwd_run(const void* gy, long long gy_ld, const float* gu, long long gu_ld, int act, float limit, int M, int inter, void* dgu, long long dgu_ld,
                         cudaStream_t stream) {
    const bool vec = inter % 8 == 0 && ok16(gy, gy_ld) && ok16(gu, gu_ld) && ok16(dgu, dgu_ld);
    const long long threads = (long long)M * (vec ? inter / 8 : inter), blocks = (threads + 255) / 256;
    if (blocks > 0x7FFFFFFFll) return ERR_TOO_LARGE;
    return (int)launch_pdl(vec ? gated_bwd_kernel<T, 8> : gated_bwd_kernel<T, 1>, dim3((unsigned)blocks), dim3(256), 0, stream, (const T*)gy, gy_ld, gu, gu_ld, act,
                           limit, (long long)M, inter, (T*)dgu, dgu_ld);
}

}  // namespace b200

using namespace b200;

static int dense_check(int dtype, int act) {
    if (dtype != F_BF16 && dtype != F_FP16) return ERR_UNSUPPORTED;
    return act < ACT_NONE || act > ACT_GELU_TANH ? ERR_UNSUPPORTED : 0;
}

// rows and columns are counted in 32 bits, a tile's overhang included
static bool too_large(int M, int N, int K) { return M > 1 << 30 || N > 1 << 30 || K > 1 << 30; }

extern "C" int b200_linear_act(const void* x, long long x_ld, const void* w, long long w_ld, int dtype, int M, int N, int K, const void* bias, int act,
                               const void* residual, long long r_ld, void* out, long long out_ld, float* z, long long z_ld, cudaStream_t stream) {
    const int rc = dense_check(dtype, act);
    if (rc) return rc;
    if (M < 0 || N <= 0 || K <= 0) return ERR_BAD_SHAPE;
    if (too_large(M, N, K)) return ERR_TOO_LARGE;
    if (M == 0) return 0;
    if (!x || !w || !out) return ERR_BAD_ARG;
    if (out_ld < N || (residual && r_ld < N) || (z && z_ld < N)) return ERR_BAD_SHAPE;
    FgArgs a{};
    a.a = {x, x_ld, 0};
    a.b = {w, w_ld, 0};
    a.M = M; a.N = N; a.K = K; a.is_f16 = dtype == F_FP16;
    a.act = act; a.bias = bias; a.res = residual; a.res_ld = r_ld; a.out = out; a.out_ld = out_ld; a.z_out = z; a.z_ld = z_ld;
    return fg_launch(a, stream);
}

extern "C" int b200_gated_linear(const void* x, long long x_ld, const void* w13, long long w_ld, int dtype, int M, int inter, int K, int act, float limit, void* out,
                                 long long out_ld, float* gu, long long gu_ld, cudaStream_t stream) {
    const int rc = dense_check(dtype, act);
    if (rc) return rc;
    if (M < 0 || inter <= 0 || inter > (1 << 29) || K <= 0 || !(limit >= 0.f)) return ERR_BAD_SHAPE;
    if (too_large(M, 2 * inter, K)) return ERR_TOO_LARGE;
    if (M == 0) return 0;
    if (!x || !w13 || !out) return ERR_BAD_ARG;
    if (out_ld < inter || (gu && gu_ld < 2 * inter)) return ERR_BAD_SHAPE;
    FgArgs a{};
    a.a = {x, x_ld, 0};
    a.b = {w13, w_ld, 0};
    a.M = M; a.N = 2 * inter; a.K = K; a.is_f16 = dtype == F_FP16;
    a.dual = 1; a.inter = inter; a.act = act; a.limit = limit; a.out = out; a.out_ld = out_ld; a.z_out = gu; a.z_ld = gu_ld;
    return fg_launch(a, stream);
}

extern "C" int b200_dense_product(const void* a_base, long long a_ld, int a_mn, const void* b_base, long long b_ld, int b_mn, int dtype, int M, int N, int K, void* out,
                                  long long out_ld, cudaStream_t stream) {
    const int rc = dense_check(dtype, 0);
    if (rc) return rc;
    if (M < 0 || N < 0 || K <= 0 || out_ld < N) return ERR_BAD_SHAPE;
    if (too_large(M, N, K)) return ERR_TOO_LARGE;
    if (M == 0 || N == 0) return 0;
    if (!a_base || !b_base || !out) return ERR_BAD_ARG;
    FgArgs a{};
    a.a = {a_base, a_ld, a_mn != 0};
    a.b = {b_base, b_ld, b_mn != 0};
    a.M = M; a.N = N; a.K = K; a.is_f16 = dtype == F_FP16;
    a.out = out; a.out_ld = out_ld;
    return fg_launch(a, stream);
}

extern "C" int b200_dense_tile(int M, int N, int K, int gated, int a_mn, int b_mn, int fp8, int has_residual, int single_values, int sms, int* tile) {
    if (M <= 0 || N <= 0 || K <= 0 || sms < 4 || !tile) return ERR_BAD_ARG;
    if (too_large(M, N, K)) return ERR_TOO_LARGE;
    FgArgs a{};
    a.a.mn_major = a_mn != 0;
    a.b.mn_major = b_mn != 0;
    a.M = M; a.N = N; a.K = fp8 ? K / 2 : K;
    a.dual = gated != 0;
    a.inter = N / 2;
    if (fp8) a.xsf = reinterpret_cast<const uint8_t*>(tile);  // what follows looks only at whether there are scales and a residual
    if (has_residual) a.res = tile;
    fg_tile(a, single_values, sms, tile);
    return 0;
}

extern "C" size_t b200_linear_act_bwd_workspace_bytes(int M, int N) {
    if (M <= 0 || N <= 0) return 0;
    return (size_t)((M + DZ_ROWS - 1) / DZ_ROWS) * (size_t)N * sizeof(float);
}

extern "C" int b200_linear_act_bwd(const void* gy, long long gy_ld, const float* z, long long z_ld, int act, int dtype, int M, int N, void* dz, long long dz_ld, void* dbias,
                                   void* workspace, size_t workspace_bytes, cudaStream_t stream) {
    const int rc = dense_check(dtype, act);
    if (rc) return rc;
    if (M < 0 || N <= 0) return ERR_BAD_SHAPE;
    if (too_large(M, N, 1)) return ERR_TOO_LARGE;
    if (act != ACT_NONE && M > 0 && !z) return ERR_BAD_ARG;
    if (M == 0) return dbias ? (int)cudaMemsetAsync(dbias, 0, (size_t)N * 2, stream) : 0;
    if (!gy || (!dz && !dbias)) return ERR_BAD_ARG;
    if (gy_ld < N || (z && z_ld < N) || (dz && dz_ld < N)) return ERR_BAD_SHAPE;
    if (dbias && (!workspace || workspace_bytes < b200_linear_act_bwd_workspace_bytes(M, N))) return ERR_WORKSPACE;
    float* part = dbias ? (float*)workspace : nullptr;
    if (act == ACT_NONE) z = nullptr;
    const int e = dtype == F_BF16 ? act_bwd_run<__nv_bfloat16>(gy, gy_ld, z, z_ld, act, M, N, dz, dz_ld, part, stream)
                                  : act_bwd_run<__half>(gy, gy_ld, z, z_ld, act, M, N, dz, dz_ld, part, stream);
    if (e || !dbias) return e;
    return column_sum(part, (M + DZ_ROWS - 1) / DZ_ROWS, N, dtype, dbias, stream);
}

extern "C" int b200_gated_linear_bwd(const void* gy, long long gy_ld, const float* gu, long long gu_ld, int act, float limit, int dtype, int M, int inter, void* dgu,
                                     long long dgu_ld, cudaStream_t stream) {
    const int rc = dense_check(dtype, act);
    if (rc) return rc;
    if (M < 0 || inter <= 0 || inter > (1 << 29) || !(limit >= 0.f)) return ERR_BAD_SHAPE;
    if (too_large(M, 2 * inter, 1)) return ERR_TOO_LARGE;
    if (M == 0) return 0;
    if (!gy || !gu || !dgu) return ERR_BAD_ARG;
    if (gy_ld < inter || gu_ld < 2 * inter || dgu_ld < 2 * inter) return ERR_BAD_SHAPE;
    return dtype == F_BF16 ? gated_bwd_run<__nv_bfloat16>(gy, gy_ld, gu, gu_ld, act, limit, M, inter, dgu, dgu_ld, stream)
                           : gated_bwd_run<__half>(gy, gy_ld, gu, gu_ld, act, limit, M, inter, dgu, dgu_ld, stream);
}

extern "C" int b200_align_rows(const void* src, long long src_ld, void* dst, long long rows, const void* src2, long long src2_ld, void* dst2, long long rows2, int cols,
                               long long dst_ld, cudaStream_t stream) {
    if (rows < 0 || rows2 < 0 || cols <= 0 || src_ld < 0 || src2_ld < 0 || dst_ld < cols) return ERR_BAD_SHAPE;
    if (rows + rows2 == 0) return 0;
    if ((rows && (!src || !dst)) || (rows2 && (!src2 || !dst2))) return ERR_BAD_ARG;
    if (((uintptr_t)src & 1) || ((uintptr_t)src2 & 1) || !ok16(dst, dst_ld) || !ok16(dst2, dst_ld)) return ERR_BAD_ALIGN;
    const long long blocks = ((rows + rows2) * ((cols + 7) / 8) + 255) / 256;
    if (blocks > 0x7FFFFFFFll) return ERR_TOO_LARGE;
    return (int)launch_pdl(align_rows_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, AlignRows{(const uint16_t*)src, src_ld, (uint16_t*)dst, rows},
                           AlignRows{(const uint16_t*)src2, src2_ld, (uint16_t*)dst2, rows2}, dst_ld, cols);
}

extern "C" size_t b200_linear_act_q8_workspace_bytes(int M, int N, int K) {
    return M <= FS_MAX_M || N <= 0 || K <= 0 ? 0 : fg_sf_workspace_bytes(M, N, K / 2);
}

extern "C" int b200_linear_act_q8(const void* x8, const void* xsf, const void* w8, const void* s8, int s_cols, int M, int N, int K, const void* bias, int act,
                                  const void* residual, long long r_ld, void* out, long long out_ld, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
    const int rc = dense_check(F_BF16, act);
    if (rc) return rc;
    if (M < 0 || N <= 0 || K <= 0 || K % 128 || s_cols < K / 32) return ERR_BAD_SHAPE;
    if (too_large(M, N, K)) return ERR_TOO_LARGE;
    if (M == 0) return 0;
    if (!x8 || !xsf || !w8 || !s8 || !out) return ERR_BAD_ARG;
    if (out_ld < N || (residual && r_ld < N)) return ERR_BAD_SHAPE;
    if (((uintptr_t)x8 & 15) || ((uintptr_t)w8 & 15) || ((uintptr_t)xsf & 3)) return ERR_BAD_ALIGN;
    FgArgs a{};
    a.a.base = x8;
    a.b.base = w8;
    a.M = M; a.N = N; a.K = K;
    a.act = act; a.bias = bias; a.res = residual; a.res_ld = r_ld; a.out = out; a.out_ld = out_ld;
    if (M <= FS_MAX_M) return fs_q8_launch(a, (const uint8_t*)xsf, (const uint8_t*)s8, s_cols, stream);
    if (!workspace || workspace_bytes < b200_linear_act_q8_workspace_bytes(M, N, K)) return ERR_WORKSPACE;
    if ((uintptr_t)workspace & 15) return ERR_BAD_ALIGN;
    a.K = K / 2;
    a.a.ld = a.b.ld = K / 2;
    a.xsf = (const uint8_t*)xsf; a.s8 = (const uint8_t*)s8; a.s_cols = s_cols;
    a.sf_workspace = workspace;
    a.sf_workspace_bytes = workspace_bytes;
    return fg_launch(a, stream);
}
