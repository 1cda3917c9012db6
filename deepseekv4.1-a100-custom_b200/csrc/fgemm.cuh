// Internal interface of the 16-bit tensor-core GEMM (fgemm.cu): bf16 x bf16 or fp16 x fp16 with fp32 accumulation.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace b200 {

// out[m, n] = epilogue( sum_k A[m, k] * B[n, k] ).  Either operand may lie with the contraction contiguous ("K-major": element (i, k) at
// base[i * ld + k]) or with its rows contiguous ("MN-major": element (i, k) at base[k * ld + i]); the tensor cores read both, so the
// products of the backward pass need no transposed copy.  Bases 16-byte aligned, ld a multiple of 8 elements.
struct FgOperand {
    const void* base;
    long long ld;
    int mn_major;
};

struct FgArgs {
    FgOperand a, b;
    int M, N, K;             // N counts the rows of B (2 * inter with dual)
    int is_f16;              // 0: bf16, 1: fp16 (operands, bias, residual and outputs)
    // epilogue: z = acc + bias;  out = act(z) + res;  z is stored too, in fp32, when z_out is given.
    // dual: B's rows are [gate | up], columns j and inter + j meet in one thread: out = act(min(g, limit)) * clamp(u, +-limit) (limit 0: no clamp);
    // z_out receives [g | u]
    int dual, inter;
    int act;
    float limit;
    const void* bias;
    const void* res;
    long long res_ld;
    void* out;
    long long out_ld;
    float* z_out;
    long long z_ld;
    // FP8 form (xsf given): A and B are e4m3 codes, their bases and K counted in pairs of codes (as the 16-bit values that TMA moves), with E8M0 scales
    // xsf [M][K/16] and s8 [ceil(N/32)][s_cols]; K a multiple of 64 pairs; bias, residual and out bf16.  sf_workspace: fg_sf_workspace_bytes, 16-byte aligned
    const uint8_t *xsf, *s8;
    int s_cols;
    void* sf_workspace;
    size_t sf_workspace_bytes;
};
size_t fg_sf_workspace_bytes(int M, int N, int K_pairs);

int fg_launch(const FgArgs& a, cudaStream_t stream);
// the kernel that a call would take on `sms` SMs: {CTAs of a tile, its columns, ways k is split}, zeros for the weight-streaming kernel; single_values: a row of the
// result, the residual or z does not start on 16 bytes
void fg_tile(const FgArgs& a, int single_values, int sms, int* tile);
// fstream.cu: the same for M <= FS_MAX_M, K-major operands
constexpr int FS_MAX_M = 16;
int fs_launch(const FgArgs& a, cudaStream_t stream);
// e4m3 operands [M][K], [N][K] (dense) with E8M0 scales xsf [M][K/32], s8 [ceil(N/32)][s_cols]; K % 128 == 0, xsf 4-byte aligned
int fs_q8_launch(const FgArgs& a, const uint8_t* xsf, const uint8_t* s8, int s_cols, cudaStream_t stream);
int fg_device_error(int* out);  // device error word (a wait that ran out of time), read and cleared

}  // namespace b200
