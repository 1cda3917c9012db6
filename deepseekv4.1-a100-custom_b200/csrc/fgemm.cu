// 16-bit GEMM on the 5th-generation tensor cores (tcgen05.mma.kind::f16, TMA, TMEM) with the epilogues of the dense operators: bias,
// activation and residual, or the gated product of two projections.
//
// Persistent CTAs, one per SM, walk the output tiles; with CG = 2 a pair of SMs (a cluster of two CTAs) shares a tile of 256 x BN
// (tcgen05 cta_group::2): each SM fetches its own 128 rows of A and half of the rows of B, so a k block costs 16 + BN/16 KB of shared memory
// traffic per 128 x BN of results where a lone SM needs 16 + BN/8.  Warp roles:
//   warp 0      TMA producer: 64-deep k blocks of both operands into a ring of shared-memory stages (128-byte swizzle)
//   warp 1      one thread (of the first CTA of a pair) issues the MMAs; the accumulators live in TMEM, two buffers, so that the epilogue of
//               a tile runs under the MMAs of the next
//   warps 4-11  epilogue: a thread owns one output row (TMEM lane) and half of the tile's columns (168 registers; 60 to 68 bytes spill)
// Every wait is bounded; one that runs out of time records a code in a device error word and the CTA runs to its end.
#include "fgemm.cuh"

#include <type_traits>

#include "common.cuh"
#include "ftypes.cuh"
#include "tc5.cuh"

namespace b200 {

__device__ int g_fg_error = 0;

constexpr int FG_THREADS = 384;
constexpr int FG_BM = 128, FG_BK = 64;  // rows of A per CTA, depth of a k block (a 128-byte row of 16-bit values)
constexpr int FG_GROUP_M = 8;           // row tiles that are walked together down the columns: their A tiles stay in L2 while B passes once
constexpr int FG_SMEM = 224 * 1024;     // ring of stages

// A stage holds two k blocks: a turn of the producer's loop costs it about 240 clocks plus 48 per copy whatever the copies' size (measured with
// copies alone), a 256 x 256 pair tile is done with a k block in 512.
// FP8 operands (MX): a k block is the same 128 bytes of a row, 128 values; a stage also holds the scale atoms of its two k blocks (tc5.cuh: 512 bytes for
// 128 rows x 4 groups of 32 k): one of A and one per 128 rows of the whole B tile.
template <int CG, int BN, bool MX>
struct FgShape {
    static constexpr uint32_t A_HALF = FG_BM * FG_BK * 2, B_ROWS = BN / CG, B_HALF = B_ROWS * FG_BK * 2, A_BYTES = 2 * A_HALF, B_BYTES = 2 * B_HALF;
    static constexpr uint32_t SFB_ATOMS = (BN + 127) / 128, SFA_BYTES = MX ? 2 * 512 : 0, SFB_BYTES = MX ? 2 * SFB_ATOMS * 512 : 0;
    static constexpr uint32_t STAGE = A_BYTES + B_BYTES + SFA_BYTES + SFB_BYTES;
    static constexpr int NS = FG_SMEM / STAGE;
    static constexpr uint32_t SF_COLS = 4 * (1 + SFB_ATOMS);  // TMEM columns of a k block's scales
    static_assert(!MX || 2 * BN + NS * 2 * SF_COLS <= 512, "accumulators and scales must fit the tensor memory");
};

struct FgParams {
    FgArgs g;
    int m_tiles, n_tiles, k_blocks;
    int split;                              // CTAs (pairs) of a cluster that share the k blocks of one tile; 1: persistent CTAs
    int vec_out, vec_res, vec_z, vec_bias;  // widest access that the rows allow: 2 = 32 bytes, 1 = 16 bytes, 0 = single values
    int turned;                             // some row allows single values only: epilogue_turned
};

template <int CG>
__device__ __forceinline__ void tc_mma_f16(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CG == 2)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(adesc), "l"(bdesc),
                     "r"(idesc), "r"(accumulate)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(adesc), "l"(bdesc),
                     "r"(idesc), "r"(accumulate)
                     : "memory");
}
// block-scaled FP8: scales of A and B in TMEM, byte j of their columns chosen by the instruction descriptor
template <int CG>
__device__ __forceinline__ void tc_mma_mx8(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    if constexpr (CG == 2)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(sfa),
            "r"(sfb)
            : "memory");
    else
        tc_mma_mx(d, adesc, bdesc, idesc, sfa, sfb, accumulate);
}
// a scale atom of shared memory into 4 TMEM columns (CG = 2: in both CTAs, each from its own shared memory)
template <int CG>
__device__ __forceinline__ void tc_cp_atom(uint32_t taddr, uint64_t sdesc) {
    if constexpr (CG == 2) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
    else tc_cp_sf(taddr, sdesc);
}
// the MMAs issued so far, when done, arrive on this barrier (CG = 2: on the barrier at the same place in both CTAs of the pair)
template <int CG>
__device__ __forceinline__ void tc_commit_pair(uint32_t bar, uint32_t lead) {
    if constexpr (CG == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)(3u << lead)) : "memory");
    else
        tc_commit(bar);
}
template <int CG>
__device__ __forceinline__ void tmem_alloc_all(uint32_t smem_dst) {
    if constexpr (CG == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_dst) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        tmem_alloc(smem_dst, 512);
        tmem_relinquish();
    }
}
template <int CG>
__device__ __forceinline__ void tmem_dealloc_all(uint32_t taddr) {
    if constexpr (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(taddr) : "memory");
    else tmem_dealloc(taddr, 512);
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// address of the same shared-memory location in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// a box into this CTA's shared memory, its bytes counted on a barrier that may lie in the other CTA of the pair
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* tm, int x, int y, uint32_t cluster_bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(tm), "r"(x), "r"(y),
                 "r"(cluster_bar)
                 : "memory");
}

// MN-major operand tile with the 128-byte swizzle: boxes of 64 rows-of-the-operand x 128 k, [box][k][64]; 8 k are 1024 bytes apart (stride
// offset), the next 64 operand rows one box further (leading offset).
__device__ __forceinline__ uint64_t desc_mn_sw128(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(16384 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// instruction descriptor of kind::f16: fp32 accumulators, both operands of one 16-bit type, M = 128
__device__ __forceinline__ uint32_t f16_idesc(int is_f16, int a_mn, int b_mn, int m, int n) {
    const uint32_t t = is_f16 ? 0u : 1u;
    return (1u << 4) | (t << 7) | (t << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

struct FgPick { int cg, bn, split; };

// instruction descriptor of kind::mxf8f6f4: both operands e4m3, K-major, E8M0 scales, byte j of the scale columns of both
__device__ __forceinline__ uint32_t mx8_idesc(int m, int n, int j) {
    return ((uint32_t)j << 4) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 4) << 24) | ((uint32_t)j << 29);
}

// a wait whose phase is usually complete already: no look at the abort flag on that path
__device__ __forceinline__ bool fg_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int where) {
    return mbar_test(bar, parity) || mbar_wait(bar, parity, abort_flag, &g_fg_error, where);
}

struct Tile { int m, n; };
__device__ __forceinline__ Tile tile_at(int i, int m_tiles, int n_tiles) {
    const int per = FG_GROUP_M * n_tiles, g = i / per, first = g * FG_GROUP_M;
    const int gm = min(FG_GROUP_M, m_tiles - first), r = i - g * per;
    return {first + r % gm, r / gm};
}

__device__ __forceinline__ void ldg32(const void* p, uint32_t (&a)[8]) {
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]), "=r"(a[4]), "=r"(a[5]), "=r"(a[6]), "=r"(a[7])
                 : "l"(p));
}
__device__ __forceinline__ void stg32(void* p, const uint32_t (&a)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(a[4]), "r"(a[5]), "r"(a[6]), "r"(a[7])
                 : "memory");
}
// 16 consecutive values of a row, of which the first n exist; a thread's row is one 32-byte sector wide here, so that the 32 rows of a warp
// cost no partial sectors
template <typename T>
__device__ __forceinline__ void load16(const T* p, int vec, int n, float (&v)[16]) {
    if (vec == 2 && n >= 16) {
        uint32_t u[8];
        ldg32(p, u);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 f = unpack2<T>(u[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    } else if (vec && n >= 16) {
        load8<T>(p, *reinterpret_cast<float(*)[8]>(&v[0]));
        load8<T>(p + 8, *reinterpret_cast<float(*)[8]>(&v[8]));
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = i < n ? to_f32(p[i]) : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void store16(T* p, int vec, int n, const float (&v)[16]) {
    if (vec == 2 && n >= 16) {
        uint32_t u[8];
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int i = 0; i < 8; ++i) u[i] = __float_as_uint(v[8 * h + i]);
                stg32(p + 8 * h, u);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
            stg32(p, u);
        }
    } else if (vec && n >= 16) {
        store8<T>(p, *reinterpret_cast<const float(*)[8]>(&v[0]));
        store8<T>(p + 8, *reinterpret_cast<const float(*)[8]>(&v[8]));
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i < n) p[i] = from_f32<T>(v[i]);
    }
}

// Bias and residual of 16 columns of a row, fetched ahead of their use (rows that allow 32-byte accesses).  For split tiles, which wait for one another
// meanwhile (64 x 4096 x 4096: 16.0 -> 15.1 us); under the products of a persistent CTA's next tile it did harm (4096 x 4096 x 2048: 58 -> 70 us).
struct Ahead { uint32_t bias[8], res[8]; bool on; };
__device__ __forceinline__ void fetch16(const FgParams& P, long long row, int col, Ahead& h) {
    const FgArgs& g = P.g;
    h.on = row < g.M && col + 16 <= g.N && (!g.bias || P.vec_bias == 2) && (!g.res || P.vec_res == 2);
    if (!h.on) return;
    if (g.bias) ldg32(reinterpret_cast<const uint16_t*>(g.bias) + col, h.bias);
    if (g.res) ldg32(reinterpret_cast<const uint16_t*>(g.res) + row * g.res_ld + col, h.res);
}

// 16 columns of one output row
template <typename T, bool AHEAD>
__device__ __forceinline__ void epilogue16(const FgParams& P, long long row, int col, const uint32_t (&acc)[16], const Ahead& h) {
    const FgArgs& g = P.g;
    const int n = g.N - col;
    float z[16], v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = __uint_as_float(acc[i]);
    auto add = [&](const void* src, const uint32_t (&ahead)[8], int vec) {
        if (AHEAD && h.on) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 f = unpack2<T>(ahead[i]);
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            }
        } else {
            load16<T>(reinterpret_cast<const T*>(src), vec, n, v);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i] += v[i];
    };
    if (g.bias) add(reinterpret_cast<const T*>(g.bias) + col, h.bias, P.vec_bias);
    if (g.z_out) store16<float>(g.z_out + row * g.z_ld + col, P.vec_z, n, z);
    act_fwd_n(g.act, z);
    if (g.res) add(reinterpret_cast<const T*>(g.res) + row * g.res_ld + col, h.res, P.vec_res);
    store16<T>(reinterpret_cast<T*>(g.out) + row * g.out_ld + col, P.vec_out, n, z);
}

// 16 columns of one row of the gated product: gate and up accumulators of output columns col ..
template <typename T>
__device__ __forceinline__ void epilogue16_dual(const FgParams& P, long long row, int col, const uint32_t (&ga)[16], const uint32_t (&ua)[16]) {
    const FgArgs& g = P.g;
    const int n = g.inter - col;
    float a[16], b[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) { a[i] = __uint_as_float(ga[i]); b[i] = __uint_as_float(ua[i]); }
    if (g.z_out) {
        float* z = g.z_out + row * g.z_ld + col;
        store16<float>(z, P.vec_z, n, a);
        store16<float>(z + g.inter, P.vec_z, n, b);
    }
    if (g.limit > 0.f) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {  // comparisons that a NaN passes through
            a[i] = a[i] > g.limit ? g.limit : a[i];
            b[i] = b[i] > g.limit ? g.limit : (b[i] < -g.limit ? -g.limit : b[i]);
        }
    }
    act_fwd_n(g.act, a);
#pragma unroll
    for (int i = 0; i < 16; ++i) a[i] *= b[i];
    store16<T>(reinterpret_cast<T*>(g.out) + row * g.out_ld + col, P.vec_out, n, a);
}

// Rows that do not start on 16 bytes (an odd width, an odd offset): a thread per row would store single values, 32 rows apart.  The warp turns its
// 32 rows x 32 accumulator columns around in shared memory and works on 32 (dual: 16) consecutive columns of a row at a time instead.
constexpr int FG_TURN_LD = 33;
constexpr int FG_TURN_BYTES = 8 * 32 * FG_TURN_LD * 4;
template <typename T>
__device__ __forceinline__ void epilogue_turned(const FgParams& P, float* buf, int lane, long long row0, int col0, const uint32_t (&a)[16], const uint32_t (&b)[16], int cols) {
    const FgArgs& g = P.g;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        buf[lane * FG_TURN_LD + i] = __uint_as_float(a[i]);
        buf[lane * FG_TURN_LD + 16 + i] = __uint_as_float(b[i]);
    }
    __syncwarp();
    // Reads of the buffer and of the residual go ahead of the stores in groups: the compiler must assume that they alias (one row at a time, a turn of 32
    // rows took 4 us).
    if (g.dual) {
        const int c = lane & 15, col = col0 + c;
        if (col >= g.inter) return;
#pragma unroll 1
        for (int r0 = lane >> 4; r0 < 32; r0 += 16) {
            float z[8], u[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                z[i] = buf[(r0 + 2 * i) * FG_TURN_LD + c];
                u[i] = buf[(r0 + 2 * i) * FG_TURN_LD + 16 + c];
            }
            const int rows = g.M - row0 - r0 < 16 ? (int)(g.M - row0 - r0) : 16;  // rows r0, r0 + 2, .. that exist: those with 2 i < rows
            if (g.z_out) {
                float* p = g.z_out + (row0 + r0) * g.z_ld + col;
#pragma unroll
                for (int i = 0; i < 8; ++i, p += 2 * g.z_ld)
                    if (2 * i < rows) {
                        p[0] = z[i];
                        p[g.inter] = u[i];
                    }
            }
            if (g.limit > 0.f) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    z[i] = z[i] > g.limit ? g.limit : z[i];
                    u[i] = u[i] > g.limit ? g.limit : (u[i] < -g.limit ? -g.limit : u[i]);
                }
            }
            act_fwd_n(g.act, z);
            T* o = reinterpret_cast<T*>(g.out) + (row0 + r0) * g.out_ld + col;
#pragma unroll
            for (int i = 0; i < 8; ++i, o += 2 * g.out_ld)
                if (2 * i < rows) *o = from_f32<T>(z[i] * u[i]);
        }
    } else {
        const int col = col0 + lane;
        if (lane >= cols || col >= g.N) return;
        const float bias = g.bias ? to_f32(reinterpret_cast<const T*>(g.bias)[col]) : 0.f;
        const int rows = g.M - row0 < 32 ? (int)(g.M - row0) : 32;
#pragma unroll 1
        for (int r0 = 0; r0 < rows; r0 += 16) {
            float z[16];
            T rv[16];
            if (g.res) {  // without a branch per row: rows behind the last one read its value
                const T* p = reinterpret_cast<const T*>(g.res) + row0 * g.res_ld + col;
#pragma unroll
                for (int i = 0; i < 16; ++i) rv[i] = p[min(r0 + i, rows - 1) * g.res_ld];
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) z[i] = buf[(r0 + i) * FG_TURN_LD + lane] + bias;
            if (g.z_out) {
                float* p = g.z_out + (row0 + r0) * g.z_ld + col;
#pragma unroll
                for (int i = 0; i < 16; ++i, p += g.z_ld)
                    if (r0 + i < rows) *p = z[i];
            }
            act_fwd_n(g.act, z);
            if (g.res)
#pragma unroll
                for (int i = 0; i < 16; ++i) z[i] += to_f32(rv[i]);
            T* o = reinterpret_cast<T*>(g.out) + (row0 + r0) * g.out_ld + col;
#pragma unroll
            for (int i = 0; i < 16; ++i, o += g.out_ld)
                if (r0 + i < rows) *o = from_f32<T>(z[i]);
        }
    }
}

template <typename T, int CG, int BN, bool A_MN, bool B_MN, bool SPLIT, bool MX>
__global__ void __launch_bounds__(FG_THREADS, 1) fg_gemm_kernel(const FgParams P, const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                                                                const __grid_constant__ CUtensorMap tm_sfa, const __grid_constant__ CUtensorMap tm_sfb) {
    using S = FgShape<CG, BN, MX>;
    constexpr int NS = S::NS;
    extern __shared__ __align__(1024) uint8_t smem_dyn[];
    __shared__ __align__(8) unsigned long long bars[2 * NS + 4];  // full[s], empty[s], acc_full[2], acc_empty[2]
    __shared__ uint32_t tmem_base_sh;
    __shared__ int abort_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t crank = CG == 2 || SPLIT ? cluster_rank() : 0;
    const uint32_t rank = crank & (CG - 1), lead = crank - rank;  // the first CTA of a pair issues the MMAs; full[] and acc_empty[] are used there
    const int slice = SPLIT ? (int)crank / CG : 0, split = SPLIT ? P.split : 1;
    uint8_t* ring = smem_dyn + ((1024u - (smem_u32(smem_dyn) & 1023u)) & 1023u);
    auto bar_full = [&](int s) { return smem_u32(&bars[s]); };
    auto bar_empty = [&](int s) { return smem_u32(&bars[NS + s]); };
    auto bar_acc_full = [&](int b) { return smem_u32(&bars[2 * NS + b]); };
    auto bar_acc_empty = [&](int b) { return smem_u32(&bars[2 * NS + 2 + b]); };
    if (tid == 0) {
        abort_flag = 0;
        for (int s = 0; s < NS; ++s) { mbar_init(bar_full(s), 1); mbar_init(bar_empty(s), 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(bar_acc_full(b), 1); mbar_init(bar_acc_empty(b), 8 * CG); }
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc_all<CG>(smem_u32(&tmem_base_sh));
    tc_fence_before();
    __syncwarp();
    if constexpr (CG == 2) cluster_sync();
    else __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_sh;
    pdl_wait();
    pdl_launch_dependents();
    const FgArgs& g = P.g;
    const int tiles = P.m_tiles * P.n_tiles, first = blockIdx.x / (CG * split), step = gridDim.x / (CG * split);
    const int n_st = (P.k_blocks + 1) / 2;  // stages of a tile; this slice's: [st_lo, st_hi)
    const int st_lo = SPLIT ? slice * n_st / split : 0, st_hi = SPLIT ? (slice + 1) * n_st / split : n_st;
    float* turn = reinterpret_cast<float*>(ring + NS * S::STAGE) + (warp & 7) * 32 * FG_TURN_LD;
    const uint32_t ring0 = smem_u32(ring), full0 = bar_full(0), empty0 = bar_empty(0);

    if (warp == 0) {
        if (lane == 0) {
            tma_prefetch_desc(&tm_a);
            tma_prefetch_desc(&tm_b);
            const uint32_t pair_full0 = CG == 2 ? map_rank(full0, lead) : full0;
            uint32_t s = 0, ph = 1, n = 0;
            for (int i = first; i < tiles && !abort_flag; i += step) {
                const Tile t = tile_at(i, P.m_tiles, P.n_tiles);
                const int m0 = (t.m * CG + (int)rank) * FG_BM;
                // the two halves of the B tile: consecutive rows, or gate rows and up rows; a CTA of a pair loads one of them
                const int h0 = g.dual ? t.n * (BN / 2) : t.n * BN, h1 = g.dual ? g.inter + h0 : h0 + BN / 2;
                const int n0 = rank ? h1 : h0;
                for (int st = st_lo; st < st_hi; ++st, ++n) {
                    if (!fg_wait(empty0 + 8 * s, ph, &abort_flag, 1)) break;
                    const uint32_t da = ring0 + s * S::STAGE, db = da + S::A_BYTES, bar = pair_full0 + 8 * s;
                    const int k0 = st * 2 * FG_BK;
                    const bool two = 2 * st + 1 < P.k_blocks;  // the last stage may hold one k block
                    if (rank == 0)
                        mbar_expect_tx(full0 + 8 * s, CG * ((A_MN || two ? S::A_BYTES : S::A_HALF) + (B_MN || two ? S::B_BYTES : S::B_HALF) + S::SFA_BYTES + S::SFB_BYTES));
                    auto load = [&](uint32_t dst, const CUtensorMap* tm, int x, int y) {
                        if constexpr (CG == 2) tma_load_2d_pair(dst, tm, x, y, bar);
                        else tma_load_2d(dst, tm, x, y, bar);
                    };
                    if constexpr (A_MN) {
#pragma unroll
                        for (int q = 0; q < FG_BM / 64; ++q) load(da + q * 16384, &tm_a, m0 + q * 64, k0);
                    } else {
                        load(da, &tm_a, k0, m0);
                        if (two) load(da + S::A_HALF, &tm_a, k0 + FG_BK, m0);
                    }
                    if constexpr (B_MN) {
#pragma unroll
                        for (int q = 0; q < (int)S::B_ROWS / 64; ++q) load(db + q * 16384, &tm_b, n0 + q * 64, k0);
                    } else {
                        load(db, &tm_b, k0, n0);
                        if constexpr (CG == 1) load(db + S::B_HALF / 2, &tm_b, k0, h1);
                        if (two) {
                            load(db + S::B_HALF, &tm_b, k0 + FG_BK, n0);
                            if constexpr (CG == 1) load(db + S::B_HALF + S::B_HALF / 2, &tm_b, k0 + FG_BK, h1);
                        }
                    }
                    if constexpr (MX) {  // atoms [128 rows][k block] and [tile][k block][SFB_ATOMS]; behind the last k block whatever follows, unused
                        load(db + S::B_BYTES, &tm_sfa, 0, (t.m * CG + (int)rank) * P.k_blocks + 2 * st);
                        load(db + S::B_BYTES + S::SFA_BYTES, &tm_sfb, 0, (t.n * P.k_blocks + 2 * st) * (int)S::SFB_ATOMS);
                    }
                    if (++s == NS) { s = 0; ph ^= 1; }
                }
            }
            // every load issued above must have landed before the CTA may exit (the second CTA of a pair is kept by the cluster barrier below)
            for (int k = 0; rank == 0 && k < NS && k < (int)n; ++k) {
                const uint32_t m = n - 1 - k, s2 = m % NS, ph2 = (m / NS) & 1;
                const unsigned long long t0 = global_timer_ns();
                while (!mbar_test(bar_full(s2), ph2))
                    if (global_timer_ns() - t0 > WAIT_LIMIT_NS) { atomicCAS(&g_fg_error, 0, 2); break; }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            const uint32_t idesc = f16_idesc(g.is_f16, A_MN, B_MN, FG_BM * CG, BN);
            const uint64_t desc_a0 = A_MN ? desc_mn_sw128(ring0) : desc_sw128(ring0);
            const uint64_t desc_b0 = B_MN ? desc_mn_sw128(ring0 + S::A_BYTES) : desc_sw128(ring0 + S::A_BYTES);
            uint32_t s = 0, ph = 0, it = 0;
            for (int i = first; i < tiles && !abort_flag; i += step, ++it) {
                const uint32_t buf = it & 1, aph = (it >> 1) & 1;
                if (!fg_wait(bar_acc_empty(buf), aph ^ 1, &abort_flag, 11)) break;
                tc_fence_after();
                const uint32_t d = tmem + buf * BN;
                for (int st = st_lo; st < st_hi; ++st) {
                    if (!fg_wait(full0 + 8 * s, ph, &abort_flag, 12)) break;
                    tc_fence_after();
                    const uint64_t da = desc_a0 + s * (S::STAGE >> 4), db = desc_b0 + s * (S::STAGE >> 4);
#pragma unroll
                    for (int j = 0; j < 2 * FG_BK / 16; ++j) {
                        if (j == FG_BK / 16 && 2 * st + 1 >= P.k_blocks) break;
                        if constexpr (MX) {  // 32 k of 8 bits are the same 32 bytes as 16 k of 16 bits
                            const uint32_t sf = tmem + 2 * BN + (s * 2 + (j >> 2)) * S::SF_COLS;
                            if ((j & 3) == 0) {
                                const uint32_t atoms = ring0 + s * S::STAGE + S::A_BYTES + S::B_BYTES + (j >> 2) * 512, atoms_b = ring0 + s * S::STAGE + S::A_BYTES + S::B_BYTES + S::SFA_BYTES + (j >> 2) * S::SFB_ATOMS * 512;
                                tc_cp_atom<CG>(sf, desc_sf_atom(atoms));
#pragma unroll
                                for (uint32_t q = 0; q < S::SFB_ATOMS; ++q) tc_cp_atom<CG>(sf + 4 + 4 * q, desc_sf_atom(atoms_b + q * 512));
                            }
                            const uint32_t o = (j & 3) * 2;
                            tc_mma_mx8<CG>(d, da + o + (j >> 2) * (S::A_HALF >> 4), db + o + (j >> 2) * (S::B_HALF >> 4), mx8_idesc(FG_BM * CG, BN, j & 3), sf, sf + 4, st != st_lo || j != 0);
                            continue;
                        }
                        // 16 k further: 32 bytes inside the swizzled row (then the second k block), or two groups of 8 k (2048 bytes)
                        const uint32_t oa = A_MN ? j * 128 : (j & 3) * 2 + (j >> 2) * (S::A_HALF >> 4), ob = B_MN ? j * 128 : (j & 3) * 2 + (j >> 2) * (S::B_HALF >> 4);
                        if constexpr (!MX) tc_mma_f16<CG>(d, da + oa, db + ob, idesc, st != st_lo || j != 0);
                    }
                    tc_commit_pair<CG>(empty0 + 8 * s, lead);
                    if (++s == NS) { s = 0; ph ^= 1; }
                }
                tc_commit_pair<CG>(bar_acc_full(buf), lead);
            }
        }
    } else if (warp >= 4) {
        const int q = warp & 3, half = warp >= 8 ? 1 : 0;
        uint32_t it = 0;
        for (int i = first; i < tiles; i += step, ++it) {
            const Tile t = tile_at(i, P.m_tiles, P.n_tiles);
            const uint32_t buf = it & 1, aph = (it >> 1) & 1;
            const long long row = (long long)(t.m * CG + (int)rank) * FG_BM + q * 32 + lane;
            if (!fg_wait(bar_acc_full(buf), aph, &abort_flag, 21)) break;
            tc_fence_after();
            if constexpr (SPLIT) break;  // the parts of the tile are added below
            const uint32_t t0 = tmem + ((uint32_t)(q * 32) << 16) + buf * BN;
            if (g.dual) {
                for (int c = half * (BN / 4); c < (half + 1) * (BN / 4); c += 16) {
                    uint32_t a[16], b[16];
                    tc_ld16(t0 + c, a);
                    tc_ld16(t0 + BN / 2 + c, b);
                    tc_wait_ld();
                    const int col = t.n * (BN / 2) + c;
                    if (P.turned) epilogue_turned<T>(P, turn, lane, row - lane, col, a, b, 16);
                    else if (row < g.M && col < g.inter) epilogue16_dual<T>(P, row, col, a, b);
                }
            } else {
                for (int c = half * (BN / 2); c < (half + 1) * (BN / 2); c += 32) {
                    uint32_t a[16], b[16];
                    tc_ld16(t0 + c, a);
                    tc_ld16(t0 + c + 16, b);
                    tc_wait_ld();
                    const int col = t.n * BN + c;
                    if (P.turned) {
                        epilogue_turned<T>(P, turn, lane, row - lane, col, a, b, 32);
                    } else if (row < g.M) {
                        if (col < g.N) epilogue16<T, false>(P, row, col, a, Ahead());
                        if (col + 16 < g.N) epilogue16<T, false>(P, row, col + 16, b, Ahead());
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (CG == 2) mbar_arrive_cluster(map_rank(bar_acc_empty(buf), lead));
                else mbar_arrive(bar_acc_empty(buf));
            }
        }
    }
    if constexpr (SPLIT) {
        // One tile per cluster, its k blocks shared by the `split` CTAs (pairs).  Each of them finishes BN / split of the columns: it gets the
        // others' accumulators of those columns in its shared memory (the ring is free by now), [slice][4 columns][row], and adds the parts
        // in slice order.
        const int W = BN / split, W2 = W / 2, nj = W / 16, n2 = g.dual ? nj / 2 : 0;
        const int q = warp & 3, half = warp >= 8 ? 1 : 0, r = q * 32 + lane;
        const uint32_t t0 = tmem + ((uint32_t)(q * 32) << 16);
        auto column = [&](int owner, int j) { return g.dual ? (j < n2 ? owner * W2 + 16 * j : BN / 2 + owner * W2 + 16 * (j - n2)) : owner * W + 16 * j; };
        const Tile t = tile_at(first, P.m_tiles, P.n_tiles);
        const long long row = (long long)(t.m * CG + (int)rank) * FG_BM + r;
        const bool some = warp >= 4 && row - lane < g.M;  // rows behind the last one are neither sent nor added
        Ahead h;
        if (some && !g.dual && !P.turned) fetch16(P, row, t.n * BN + slice * W + 16 * half, h);  // under the exchange
        __syncwarp();
        cluster_sync();  // every CTA's MMAs have read their stages
        tc_fence_after();
        if (some) {
            for (int o = 0; o < split; ++o) {
                if (o == slice) continue;
                const uint32_t dst = map_rank(smem_u32(ring), (uint32_t)(o * CG) + rank) + (uint32_t)(slice * (W / 4) * FG_BM + r) * 16u;
                for (int j = half; j < nj; j += 2) {
                    uint32_t a[16];
                    tc_ld16(t0 + column(o, j), a);
                    tc_wait_ld();
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + (uint32_t)((4 * j + i) * FG_BM) * 16u), "r"(a[4 * i]), "r"(a[4 * i + 1]),
                                     "r"(a[4 * i + 2]), "r"(a[4 * i + 3])
                                     : "memory");
                }
            }
        }
        __syncwarp();
        cluster_sync();
        if (some) {
            auto sum16 = [&](int j, uint32_t (&out)[16]) {
                uint32_t a[16];
                tc_ld16(t0 + column(slice, j), a);
                tc_wait_ld();
                float v[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = 0.f;
                for (int sl = 0; sl < split; ++sl) {
                    if (sl == slice) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] += __uint_as_float(a[i]);
                    } else {
                        const float4* src = reinterpret_cast<const float4*>(ring) + (sl * (W / 4) + 4 * j) * FG_BM + r;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float4 f = src[i * FG_BM];
                            v[4 * i] += f.x; v[4 * i + 1] += f.y; v[4 * i + 2] += f.z; v[4 * i + 3] += f.w;
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) out[i] = __float_as_uint(v[i]);
            };
            if (g.dual) {
                for (int j = half; j < n2; j += 2) {
                    uint32_t a[16], b[16];
                    sum16(j, a);
                    sum16(n2 + j, b);
                    const int col = t.n * (BN / 2) + slice * W2 + 16 * j;
                    if (P.turned) epilogue_turned<T>(P, turn, lane, row - lane, col, a, b, 16);
                    else if (row < g.M && col < g.inter) epilogue16_dual<T>(P, row, col, a, b);
                }
            } else {
                for (int j = half; j < nj; j += 2) {
                    uint32_t a[16];
                    sum16(j, a);
                    const int col = t.n * BN + slice * W + 16 * j;
                    if (P.turned) epilogue_turned<T>(P, turn, lane, row - lane, col, a, a, 16);
                    else if (row < g.M && col < g.N) epilogue16<T, true>(P, row, col, a, h);
                    if (!P.turned && j + 2 < nj) fetch16(P, row, col + 32, h);
                }
            }
        }
    }
    tc_fence_before();
    __syncwarp();
    if constexpr (CG == 2) cluster_sync();  // neither CTA of a pair leaves while the other may still signal its barriers or read its tensor memory
    else __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_all<CG>(tmem);
    }
}

// ------------------------------------------------------------------ host
int sm_count();

static int fg_tmap(CUtensorMap* tm, const FgOperand& o, int is_f16, long long rows, long long k, uint32_t box_rows) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return (int)cudaErrorNotSupported;
    cuuint64_t dims[2] = {(cuuint64_t)(o.mn_major ? rows : k), (cuuint64_t)(o.mn_major ? k : rows)};
    cuuint64_t strides[1] = {(cuuint64_t)o.ld * 2};
    cuuint32_t box[2] = {64, o.mn_major ? 2u * FG_BK : box_rows};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(tm, is_f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(o.base), dims, strides, box, estr,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : (int)cudaErrorInvalidValue;
}

// scale atoms as rows of 128 words, read `atoms` rows at a time
static int fg_sf_tmap(CUtensorMap* tm, const void* base, long long rows, uint32_t atoms) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return (int)cudaErrorNotSupported;
    cuuint64_t dims[2] = {128, (cuuint64_t)rows};
    cuuint64_t strides[1] = {512};
    cuuint32_t box[2] = {128, atoms}, estr[2] = {1, 1};
    CUresult r = fn(tm, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : (int)cudaErrorInvalidValue;
}

// E8M0 scales into atom order, one block of 128 threads per atom: byte (r % 32) * 16 + (r / 32) * 4 + g of an atom = scale of row r, group g of the
// k block.  Atoms of x: [128 rows][k block], one row of scales per row; atoms of w: [tile of bn rows][k block][ceil(bn / 128)], one row of scales per
// 32 rows.  Rows behind the last one borrow its scales (their products are not stored).
__global__ void __launch_bounds__(128) fg_scale_atoms_kernel(const uint8_t* __restrict__ xsf, int M, const uint8_t* __restrict__ s8, int s_cols, int N, int k_blocks, int bn,
                                                             int x_atoms, uint32_t* __restrict__ out) {
    pdl_wait();
    pdl_launch_dependents();
    const int atom = blockIdx.x, r = threadIdx.x;
    const uint8_t* src;
    if (atom < x_atoms) {
        const int mt = atom / k_blocks, kb = atom - mt * k_blocks;
        src = xsf + (long long)min(mt * 128 + r, M - 1) * (k_blocks * 4) + kb * 4;
    } else {
        const int per = (bn + 127) / 128, i = atom - x_atoms, tk = i / per, nt = tk / k_blocks, kb = tk - nt * k_blocks;
        src = s8 + (long long)(min(nt * bn + (i - tk * per) * 128 + r, N - 1) >> 5) * s_cols + kb * 4;
    }
    out[(long long)atom * 128 + (r & 31) * 4 + (r >> 5)] = src[0] | src[1] << 8 | src[2] << 16 | (uint32_t)src[3] << 24;
}

template <typename T, int CG, int BN, bool A_MN, bool B_MN, bool SPLIT, bool MX>
static int fg_run(FgParams& P, cudaStream_t stream) {
    using S = FgShape<CG, BN, MX>;
    const FgArgs& g = P.g;
    P.m_tiles = (g.M + CG * FG_BM - 1) / (CG * FG_BM);
    P.n_tiles = g.dual ? (g.inter + BN / 2 - 1) / (BN / 2) : (g.N + BN - 1) / BN;
    P.k_blocks = (g.K + FG_BK - 1) / FG_BK;
    if ((long long)P.m_tiles * P.n_tiles > 0x0FFFFFFFll) return ERR_TOO_LARGE;
    alignas(64) CUtensorMap ta, tb, tsa, tsb;
    int rc = fg_tmap(&ta, g.a, g.is_f16, g.M, g.K, FG_BM);
    if (!rc) rc = fg_tmap(&tb, g.b, g.is_f16, g.N, g.K, BN / 2);
    tsa = tsb = ta;
    if constexpr (MX) {
        const long long xa = (long long)((g.M + 127) / 128) * P.k_blocks, wa = (long long)P.n_tiles * P.k_blocks * S::SFB_ATOMS;
        if (xa + wa > 0x7FFFFFFFll) return ERR_TOO_LARGE;
        if ((size_t)(xa + wa) * 512 > g.sf_workspace_bytes) return ERR_WORKSPACE;
        if (!rc) rc = fg_sf_tmap(&tsa, g.sf_workspace, xa, 2);
        if (!rc) rc = fg_sf_tmap(&tsb, (const uint8_t*)g.sf_workspace + xa * 512, wa, 2 * S::SFB_ATOMS);
        if (rc) return rc;
        const cudaError_t e = launch_pdl(fg_scale_atoms_kernel, dim3((unsigned)(xa + wa)), dim3(128), 0, stream, g.xsf, g.M, g.s8, g.s_cols, g.N, P.k_blocks, BN, (int)xa,
                                         (uint32_t*)g.sf_workspace);
        if (e != cudaSuccess) return (int)e;
    }
    if (rc) return rc;
    const size_t smem = (size_t)S::NS * S::STAGE + 1024 + (P.turned ? FG_TURN_BYTES : 0);
    constexpr int smem_max = S::NS * S::STAGE + 1024 + (BN == 192 || MX ? 0 : FG_TURN_BYTES);
    auto kernel = fg_gemm_kernel<T, CG, BN, A_MN, B_MN, SPLIT, MX>;
    static bool attr_done[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !attr_done[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_max);
        if (e != cudaSuccess) return (int)e;
        if (dev >= 0 && dev < 64) attr_done[dev] = true;
    }
    const int tiles = P.m_tiles * P.n_tiles, groups = sm_count() / CG, cluster = CG * P.split;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(SPLIT ? tiles * cluster : (tiles < groups ? tiles : groups) * CG);
    cfg.blockDim = dim3(FG_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return (int)cudaLaunchKernelEx(&cfg, kernel, P, ta, tb, tsa, tsb);
}

template <typename T, int CG, int BN, bool SPLIT>
static int fg_layouts(FgParams& P, cudaStream_t stream) {
    if constexpr (BN != 256 && std::is_same<T, __nv_bfloat16>::value) {
        if (P.g.xsf) return fg_run<T, CG, BN, false, false, SPLIT, true>(P, stream);
    }
    if (P.g.xsf) return ERR_UNSUPPORTED;
    if constexpr (BN == 192) {  // MN-major boxes are 64 rows wide: a pair's 96 rows of B are no multiple of that
        return P.g.b.mn_major || P.g.a.mn_major ? ERR_UNSUPPORTED : fg_run<T, CG, BN, false, false, SPLIT, false>(P, stream);
    } else {
        if (P.g.a.mn_major) return P.g.b.mn_major ? fg_run<T, CG, BN, true, true, SPLIT, false>(P, stream) : ERR_UNSUPPORTED;
        return P.g.b.mn_major ? fg_run<T, CG, BN, false, true, SPLIT, false>(P, stream) : fg_run<T, CG, BN, false, false, SPLIT, false>(P, stream);
    }
}

// Which tile, and how many ways its k is split.  Each choice's time is estimated as (turns of the busiest CTA) x (time of a tile: its stages' products, or
// its epilogue where that is longer) + (start, end and last epilogue), the constants in us from measurements over 25 shapes between 64 x 4096 x 2048 and
// 8192 x 8192 x 8192; e.g. measured 64 x 4096 x 4096: 1/128/4 13.9, 1/128/1 20.9, 2/256/1 25.7; 512 x 4096 x 4096: 2/256/2 21.3, 1/128/1 22.0,
// 1/128/4 47.5; 1500 x 4096 x 4096: 2/192/1 41.9, 2/256/1 48.0, 1/128/1 55.9; 4096 x 12288 x 4096: 2/256/1 275, 2/192/1 290, 1/128/1 384 (single products on a
// cool device; the last one takes 303 in a loop with gelu and 351 among other work, under the 1000 W limit).
// FP8: 64 x 4096 x 4096: 1/128/4 14.4, 1/128/1 19.5, 2/192/1 24.1; 4096 x 12288 x 4096: 2/192/1 202, 1/128/1 249; 4096 x 4096 x 2048: 2/192/1 47 and with a
// residual 55, where the estimate is 39 and 43.
// 128-column tiles of a pair are not compiled: they cost what 128 x 128 tiles of one SM cost or more, in as many turns or more.
static FgPick fg_pick(const FgParams& P, int sms) {
    const FgArgs& g = P.g;
    static const struct { FgPick k; double stage, stage_mx, fixed, epi, epi_res; } choices[] = {
        {{1, 128, 1}, .54, .76, 4.0, 2.5, 4.8},  {{1, 128, 2}, .54, .69, 7.5, 0, 0},    {{1, 128, 4}, .54, .69, 8.5, 0, 0},
        {{2, 192, 1}, .645, .83, 5.5, 4.2, 7.5}, {{2, 256, 1}, .78, 0, 6.5, 5.0, 9.0}, {{2, 256, 2}, .78, 0, 10.0, 0, 0}};
    const int st = (g.K + 2 * FG_BK - 1) / (2 * FG_BK);
    FgPick best{1, 128, 1};
    double best_t = 1e30;
    for (const auto& c : choices) {
        const FgPick& k = c.k;
        if (k.split > st || (k.bn == 192 && (g.a.mn_major || g.b.mn_major || P.turned)) || (k.bn == 256 && g.xsf)) continue;
        const int cols = g.dual ? k.bn / 2 : k.bn, width = g.dual ? g.inter : g.N;
        const long long tiles = ((long long)g.M + k.cg * FG_BM - 1) / (k.cg * FG_BM) * ((width + cols - 1) / cols);
        const int groups = sms / (k.cg * k.split);
        const double turns = (double)((tiles + groups - 1) / groups), stage = g.xsf ? c.stage_mx : c.stage, epi = g.res ? c.epi_res : c.epi;
        // persistent CTAs pay the fixed part once, clusters that split a tile once per turn
        const double t = k.split > 1 ? turns * ((st + k.split - 1) / k.split * stage + c.fixed) : turns * (st * stage > epi ? st * stage : epi) + c.fixed;
        if (t < best_t) { best_t = t; best = k; }
    }
    return best;
}

template <typename T>
static int fg_dispatch(FgParams& P, cudaStream_t stream) {
    const FgPick k = fg_pick(P, sm_count());
    P.split = k.split;
    if (k.cg == 1) return k.split > 1 ? fg_layouts<T, 1, 128, true>(P, stream) : fg_layouts<T, 1, 128, false>(P, stream);
    if (k.bn == 192) return fg_layouts<T, 2, 192, false>(P, stream);
    return k.split > 1 ? fg_layouts<T, 2, 256, true>(P, stream) : fg_layouts<T, 2, 256, false>(P, stream);
}

// the products of up to FS_MAX_M rows with K-major 16-bit operands are fstream.cu's
static bool fg_streams(const FgArgs& a) { return a.M <= FS_MAX_M && !a.a.mn_major && !a.b.mn_major && !a.xsf; }

void fg_tile(const FgArgs& a, int single_values, int sms, int* tile) {
    FgParams P{};
    P.g = a;
    P.turned = !a.xsf && single_values;
    const FgPick k = a.M <= FS_MAX_M && (a.xsf || fg_streams(a)) ? FgPick{0, 0, 0} : fg_pick(P, sms);
    tile[0] = k.cg; tile[1] = k.bn; tile[2] = k.split;
}

int fg_launch(const FgArgs& a, cudaStream_t stream) {
    if (!a.a.base || !a.b.base || !a.out) return ERR_BAD_ARG;
    if (a.M <= 0 || a.N <= 0 || a.K <= 0) return ERR_BAD_SHAPE;
    if (a.dual && (a.N != 2 * a.inter || a.b.mn_major)) return ERR_BAD_SHAPE;
    if (((uintptr_t)a.a.base & 15) || ((uintptr_t)a.b.base & 15) || a.a.ld % 8 || a.b.ld % 8) return ERR_BAD_ALIGN;
    if (a.a.ld < (a.a.mn_major ? a.M : a.K) || a.b.ld < (a.b.mn_major ? a.N : a.K)) return ERR_BAD_SHAPE;
    if (fg_streams(a)) return fs_launch(a, stream);
    FgParams P{};
    P.g = a;
    auto vec = [](const void* p, long long ld_bytes) {
        const uintptr_t u = (uintptr_t)p | (uintptr_t)ld_bytes;
        return u & 15 ? 0 : (u & 31 ? 1 : 2);
    };
    P.vec_out = vec(a.out, a.out_ld * 2);
    P.vec_res = vec(a.res, a.res_ld * 2);
    P.vec_z = vec(a.z_out, a.dual ? a.z_ld * 4 | a.inter * 4 : a.z_ld * 4);
    P.vec_bias = vec(a.bias, 0);
    // FP8 has no room for the turning buffer: its single values are stored 32 rows apart (4096 x 4097 x 2048 with residual 197 us, 4096 x 4096 x 2048 55)
    P.turned = !a.xsf && (!P.vec_out || (a.res && !P.vec_res) || (a.z_out && !P.vec_z));
    return a.is_f16 ? fg_dispatch<__half>(P, stream) : fg_dispatch<__nv_bfloat16>(P, stream);
}

size_t fg_sf_workspace_bytes(int M, int N, int K_pairs) {
    const size_t kb = (K_pairs + FG_BK - 1) / FG_BK, x = ((size_t)M + 127) / 128, w128 = ((size_t)N + 127) / 128, w192 = ((size_t)N + 191) / 192 * 2;
    return (x + (w128 > w192 ? w128 : w192)) * kb * 512;
}

int fg_device_error(int* out) {
    int v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, g_fg_error, sizeof(int));
    if (e != cudaSuccess) return (int)e;
    if (v) {
        int z = 0;
        cudaMemcpyToSymbol(g_fg_error, &z, sizeof(int));
    }
    *out = v;
    return 0;
}

}  // namespace b200
