// g1_gated.cuh -- the gated feed-forward layer on the tensor cores (tcgen05), forward and backward:
//
//   g = X Wg^T + bg,  u = X Wu^T + bu,  h = act(g) * u          X [M][K], W [2F][K] = [Wg; Wu], b [2F]
//   dg = dh u act'(g),  du = dh act(g)
//   dX = dg Wg + du Wu,   dWg = dg^T X,  dWu = du^T X,   dbg = sum over rows of dg,  dbu = sum of du
//
// X, W, h and their gradients are bf16 or fp16, sums and everything between the products fp32; h, dX and dW are
// rounded once.  dg and du are rounded to the 16-bit type between the two backward products (they are
// operands of the tensor cores there): half a step of each term, which averages over the sum and stays below
// the result's own rounding; db is summed from the unrounded values.
//
// One kernel, k_ff, in four modes, all C = A B over 128 x BN tiles with fp32 accumulators in tensor memory:
//
//   FWD  A = X, B = 128 rows of Wg and the same 128 rows of Wu, one MMA of N = 256; the epilogue holds g and u of
//        128 outputs side by side and writes h.  Neither g nor u leaves the SM.
//   DZ   the same product again; the epilogue reads dh and writes z = [dg | du] ([M][2 Fp]) and the column
//        sums.  Recomputing g and u costs 4MKF operations of the backward's 12MKF; keeping them at the accuracy
//        that db needs (fp32) would write and read 16 bytes an output, more time than the product up to K = 1024
//        or so, and hold 8 bytes an output between forward and backward.
//   DX   A = z, B = W read along its rows (MN-major): no transposed copy.
//   DW   A = z^T, B = X^T, both MN-major straight from their row-major tiles, summed over M.  The 2F x K tiles are
//        few and M is long: see the work split at k_ff's iterator.
//
// Operands come by TMA (128-byte swizzle, zero fill past the edges, no multicast) in chunks of 64 along the sum,
// four stages; one thread issues the loads, one the MMAs, sixteen warps run the epilogue of a tile while the
// next one accumulates in the other half of tensor memory.  Every wait is bounded; one that runs out sets g_err
// (g1_gated_ff_status), and the kernel ends with garbage in its outputs.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace g1ff {

using g1gemm::s32;
using g1gemm::tma_load_2d;

constexpr int BM = 128, BK = 64, STAGES = 4, EPI_WARPS = 16, NTH = 64 + 32 * EPI_WARPS;
enum { FWD = 0, DZ = 1, DX = 2, DW = 3 };
constexpr int DW_BLOCK = 64;  // chunks (of 64 rows) that the CTAs of DW walk together

__device__ int g_err;  // a wait ran out

struct Args {
    CUtensorMap a0, a1, b0, b1;  // gate / up halves where they differ
    int M, N, nk;                // rows and columns of the output (FWD, DZ: N = F); chunks of the sum
    int F, act;
    const float* bias;           // [2F] or null
    const void* dh;              // DZ: [M][F]
    void* out;                   // h [M][F], z [M][2 Fp], dX [M][K], or the fp32 partial tiles
    long long ldo;
    float* db;                   // DZ: [gridDim][4][2F] column sums, zeroed, or null
    int tile0, ntp;              // DW: the pass's tiles
    int vec;                     // rows of the output (and of dh) are 16-byte aligned
};

__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity) {
    const uint32_t a = s32(bar);
    for (uint32_t it = 0; it < g1gemm::SPIN; ++it) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(a), "r"(parity)
            : "memory");
        if (done) return true;
    }
    return false;
}

// MN-major SWIZZLE_128B descriptor of 64 x 64 boxes 8 KB apart: LBO = the next 64 along M or N, SBO = the next 8
// along the sum (8 rows of 128 bytes)
__device__ __forceinline__ uint64_t desc_mn(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(8192 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) |
           (2ull << 61);
}

template <class T>
struct Half2;
template <>
struct Half2<__nv_bfloat16> {
    static constexpr uint32_t fmt = 1;
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t v) {
        return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
    }
    static __device__ __forceinline__ __nv_bfloat16 one(float a) { return __float2bfloat16_rn(a); }
    static __device__ __forceinline__ float f(__nv_bfloat16 a) { return __bfloat162float(a); }
};
template <>
struct Half2<__half> {
    static constexpr uint32_t fmt = 0;
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
    static __device__ __forceinline__ __half one(float a) { return __float2half_rn(a); }
    static __device__ __forceinline__ float f(__half a) { return __half2float(a); }
};

__device__ __forceinline__ float sigmoid(float g) {
    float r;
    asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.f + __expf(-g)));
    return r;
}

// act(g) and, with D, act'(g)
template <int ACT, bool D>
__device__ __forceinline__ void act1(float g, float& a, float& d) {
    if (ACT == 0) {
        a = tanhf(g);
        if (D) d = 1.f - a * a;
    } else if (ACT == 1) {
        const float e = expm1f(fminf(g, 0.f));
        a = g > 0.f ? g : e;
        if (D) d = g > 0.f ? 1.f : e + 1.f;
        if (g != g) a = d = g;  // fminf drops a NaN
    } else if (ACT == 2) {
        const float s = sigmoid(g);
        a = g * s;
        if (D) d = fmaf(a, 1.f - s, s);
    } else {
        const float c = fmaf(0.5f, erff(g * 0.70710678118654752f), 0.5f);
        a = g * c;
        if (D) d = fmaf(g * 0.39894228040143268f, __expf(-0.5f * g * g), c);
    }
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

template <int BN>
struct Smem {
    uint8_t a[STAGES][BM * BK * 2];
    uint8_t b[STAGES][BN * BK * 2];
    uint64_t full[STAGES], empty[STAGES], tfull[2], tempty[2];
    uint32_t tslot;
    volatile int stop;  // a wait of this CTA ran out
};
template <int BN>
constexpr int smem_bytes() { return (int)sizeof(Smem<BN>) + 1024; }

// 16 values of a row to 16-bit memory, `n` of them inside the matrix
template <class T>
__device__ __forceinline__ void store16(T* dst, const float* v, int n, bool vec) {
    if (vec && n >= 16) {
        uint32_t pk[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) pk[j] = Half2<T>::pack(v[2 * j], v[2 * j + 1]);
        reinterpret_cast<uint4*>(dst)[0] = make_uint4(pk[0], pk[1], pk[2], pk[3]);
        reinterpret_cast<uint4*>(dst)[1] = make_uint4(pk[4], pk[5], pk[6], pk[7]);
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (j < n) dst[j] = Half2<T>::one(v[j]);
    }
}

__device__ __forceinline__ void load_bias(const float* bias, int n, float* v) {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = (bias && j < n) ? __ldg(bias + j) : 0.f;
}

template <class T>
__device__ __forceinline__ void load16(const T* src, float* v, int n, bool vec) {
    if (vec && n >= 16) {
        const uint4 a = __ldcs(reinterpret_cast<const uint4*>(src)), b = __ldcs(reinterpret_cast<const uint4*>(src) + 1);
        const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float2 f = Half2<T>::unpack(w[j]);
            v[2 * j] = f.x;
            v[2 * j + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = j < n ? Half2<T>::f(src[j]) : 0.f;
    }
}

// lane l gets the sum over the warp's lanes of v[l]: halves of the list change sides 5 times (31 shuffles)
__device__ __forceinline__ float column_sums(float (&v)[32], int lane) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const bool up = lane & o;
#pragma unroll
        for (int j = 0; j < o; ++j) {
            const float send = up ? v[j] : v[j + o], keep = up ? v[j + o] : v[j];
            v[j] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
    }
    return v[0];
}

template <class T, int ACT>
__device__ __forceinline__ void fwd16(const uint32_t* rg, const uint32_t* ru, const float* bg, const float* bu, float* h) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        float a, d;
        act1<ACT, false>(__uint_as_float(rg[j]) + bg[j], a, d);
        h[j] = a * (__uint_as_float(ru[j]) + bu[j]);
    }
}
template <class T, int ACT>
__device__ __forceinline__ void dz16(const uint32_t* rg, const uint32_t* ru, const float* bg, const float* bu,
                                     const float* dh, float* z) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        float a, d;
        act1<ACT, true>(__uint_as_float(rg[j]) + bg[j], a, d);
        z[j] = dh[j] * (__uint_as_float(ru[j]) + bu[j]) * d;
        z[16 + j] = dh[j] * a;
    }
}

// The tiles of a CTA.  FWD, DZ, DX: 128-row blocks by column tiles, columns fastest, so that the CTAs in flight
// share rows of A in L2 and A comes from HBM once (the weights stay in L2).
// DW: the sum over M is cut for the CTAs to be equally loaded, each CTA keeping at most two tiles (two
// accumulators) from start to end: rows are walked in blocks of DW_BLOCK chunks, and of each block's ntp x DW_BLOCK
// (tile, chunk) units CTA b takes the same b-th share.  All CTAs stay within a block of rows, so X and z come from HBM
// once; cutting each tile's whole M into runs instead would have the tiles read the same rows at different times.
template <int MODE>
struct Tiles {
    int tile, step, count, acc;      // FWD, DZ, DX
    int t0, c0, c1, c2, blk;         // DW: chunks [c0, c1) of tile t0 and [0, c2) of tile t0 + 1 in each block
    __device__ __forceinline__ Tiles(const Args& P, int ntiles) {
        if (MODE == DW) {
            blk = min(DW_BLOCK, P.nk);
            const long long U = (long long)P.ntp * blk;
            const long long u0 = U * blockIdx.x / gridDim.x, u1 = U * (blockIdx.x + 1) / gridDim.x;
            t0 = (int)(u0 / blk);
            c0 = (int)(u0 % blk);
            c1 = (int)min((long long)blk, c0 + (u1 - u0));
            c2 = (int)(u1 - u0) - (c1 - c0);
        } else {
            tile = blockIdx.x;
            step = gridDim.x;
            count = ntiles;
        }
    }
};

template <class T, int MODE, int BN>
__global__ void __launch_bounds__(NTH, 1) k_ff(const __grid_constant__ Args P) {
    extern __shared__ uint8_t smem_raw[];
    Smem<BN>& S = *reinterpret_cast<Smem<BN>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    constexpr bool A_MN = MODE == DW, B_MN = MODE == DX || MODE == DW, PAIR = MODE == FWD || MODE == DZ;
    constexpr int TN = PAIR ? BN / 2 : BN;  // output columns a tile
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int ntn = (P.N + TN - 1) / TN;
    // DW: row tiles of the gate half, then of the up half
    const int half_tiles = (P.F + BM - 1) / BM;
    const int ntm = MODE == DW ? 2 * half_tiles : (P.M + BM - 1) / BM;
    const int ntiles = ntm * ntn, nk = P.nk;
    if (tid == 0) {
        S.stop = 0;
        for (int i = 0; i < STAGES; ++i) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(s32(&S.full[i])));
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(s32(&S.empty[i])));
        }
        for (int i = 0; i < 2; ++i) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(s32(&S.tfull[i])));
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(s32(&S.tempty[i])), "r"(EPI_WARPS));
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(&S.tslot)), "r"(2 * BN));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;");
    const uint32_t tmem = S.tslot;
    bool ok = true;
    const Tiles<MODE> W(P, ntiles);

    if (warp == 0 && lane == 0) {  // loads
        int stage = 0;
        uint32_t phase = 0;
        auto load = [&](int tile, int c) -> bool {
            if (!wait(&S.empty[stage], phase ^ 1u)) return false;
            uint64_t* bar = &S.full[stage];
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(s32(bar)), "r"((BM + BN) * BK * 2)
                         : "memory");
            const int mt = tile / ntn, n0 = (tile % ntn) * TN;
            uint8_t *as = S.a[stage], *bs = S.b[stage];
            if (PAIR) {
                tma_load_2d(as, &P.a0, c * BK, mt * BM, bar);
                tma_load_2d(bs, &P.b0, c * BK, n0, bar);
                tma_load_2d(bs + TN * BK * 2, &P.b1, c * BK, n0, bar);
            } else if (MODE == DX) {
                // the sum runs over the gate half's columns, then the up half's
                const bool up = c >= nk / 2;
                const int k0 = (up ? c - nk / 2 : c) * BK;
                tma_load_2d(as, up ? &P.a1 : &P.a0, k0, mt * BM, bar);
#pragma unroll
                for (int j = 0; j < BN / 64; ++j) tma_load_2d(bs + j * 8192, up ? &P.b1 : &P.b0, n0 + 64 * j, k0, bar);
            } else {
                const bool up = mt >= half_tiles;
                const int f0 = (up ? mt - half_tiles : mt) * BM;
#pragma unroll
                for (int j = 0; j < BM / 64; ++j) tma_load_2d(as + j * 8192, up ? &P.a1 : &P.a0, f0 + 64 * j, c * BK, bar);
#pragma unroll
                for (int j = 0; j < BN / 64; ++j) tma_load_2d(bs + j * 8192, &P.b0, n0 + 64 * j, c * BK, bar);
            }
            if (++stage == STAGES) { stage = 0; phase ^= 1u; }
            return true;
        };
        if (MODE == DW) {
            for (int base = 0; base < nk && ok; base += W.blk) {
                for (int c = W.c0; c < W.c1 && ok; ++c)
                    if (base + c < nk) ok = load(P.tile0 + W.t0, base + c);
                for (int c = 0; c < W.c2 && ok; ++c)
                    if (base + c < nk) ok = load(P.tile0 + W.t0 + 1, base + c);
            }
        } else {
            for (int tile = W.tile; tile < ntiles && ok; tile += W.step)
                for (int c = 0; c < nk && ok; ++c) ok = load(tile, c);
        }
    } else if (warp == 1 && lane == 0) {  // MMAs
        constexpr uint32_t idesc = (1u << 4) | (Half2<T>::fmt << 7) | (Half2<T>::fmt << 10) | ((A_MN ? 1u : 0u) << 15) |
                                   ((B_MN ? 1u : 0u) << 16) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
        int stage = 0;
        uint32_t phase = 0;
        auto mma = [&](uint32_t d, bool first) -> bool {
            if (!wait(&S.full[stage], phase)) return false;
            asm volatile("tcgen05.fence::after_thread_sync;");
            const uint32_t a0 = s32(S.a[stage]), b0 = s32(S.b[stage]);
#pragma unroll
            for (int k = 0; k < BK / 16; ++k) {
                const uint64_t ad = A_MN ? desc_mn(a0 + k * 2048) : g1gemm::desc_sw128(a0 + k * 32);
                const uint64_t bd = B_MN ? desc_mn(b0 + k * 2048) : g1gemm::desc_sw128(b0 + k * 32);
                const uint32_t accum = (!first || k > 0) ? 1u : 0u;
                asm volatile(
                    "{\n\t.reg .pred p;\n\t"
                    "setp.ne.b32 p, %4, 0;\n\t"
                    "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
                    "l"(ad), "l"(bd), "r"(idesc), "r"(accum));
            }
            asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                             s32(&S.empty[stage]))
                         : "memory");
            if (++stage == STAGES) { stage = 0; phase ^= 1u; }
            return true;
        };
        auto commit = [&](int acc) {
            asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                             s32(&S.tfull[acc]))
                         : "memory");
        };
        if (MODE == DW) {
            for (int base = 0; base < nk && ok; base += W.blk) {
                for (int c = W.c0; c < W.c1 && ok; ++c)
                    if (base + c < nk) ok = mma(tmem, base == 0 && c == W.c0);
                for (int c = 0; c < W.c2 && ok; ++c)
                    if (base + c < nk) ok = mma(tmem + BN, base == 0 && c == 0);
            }
            if (ok) { commit(0); commit(1); }
        } else {
            uint32_t acc = 0, accph = 0;
            for (int tile = W.tile; tile < ntiles && ok; tile += W.step) {
                if (!wait(&S.tempty[acc], accph ^ 1u)) { ok = false; break; }
                asm volatile("tcgen05.fence::after_thread_sync;");
                for (int c = 0; c < nk && ok; ++c) ok = mma(tmem + acc * BN, c == 0);
                if (ok) commit(acc);
                if (++acc == 2) { acc = 0; accph ^= 1u; }
            }
        }
    } else if (warp >= 2) {  // epilogue: warp w reads TMEM lanes 32 (w & 3) .., part (w - 2) / 4 of the columns
        const int q = warp & 3, part = (warp - 2) >> 2;
        constexpr int CW = TN / 4;
        static_assert(CW % 16 == 0, "16-column TMEM loads");
        const uint32_t tl = tmem + ((uint32_t)(32 * q) << 16);
        if (MODE == DW) {
            // fp32 partial tiles, row-major [128][BN]; slot b + t is this CTA's alone (a next share raises b or t)
            for (int a = 0; a < 2 && ok; ++a) {
                const bool have = a == 0 ? W.c1 > W.c0 : W.c2 > 0;
                if (!have) continue;
                // all of the CTA's products lie before this: as long as 64 other waits, or until one of those ran out
                ok = false;
                for (int i = 0; i < 64 && !ok && !S.stop; ++i) ok = wait(&S.tfull[a], 0);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;");
                float* dst = (float*)P.out + ((size_t)(blockIdx.x + W.t0 + a) * BM + 32 * q + lane) * BN + part * CW;
#pragma unroll 1
                for (int cc = 0; cc < CW; cc += 16) {
                    uint32_t r[16];
                    tmem_ld16(tl + a * BN + part * CW + cc, r);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        reinterpret_cast<uint4*>(dst + cc)[j] = make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
                }
            }
        } else {
            uint32_t acc = 0, accph = 0;
            for (int tile = W.tile; tile < ntiles; tile += W.step) {
                if (!wait(&S.tfull[acc], accph)) { ok = false; break; }
                asm volatile("tcgen05.fence::after_thread_sync;");
                const int row = (tile / ntn) * BM + 32 * q + lane, n0 = (tile % ntn) * TN + part * CW;
                const uint32_t t0 = tl + acc * BN + part * CW;
#pragma unroll 1
                for (int cc = 0; cc < CW; cc += 16) {
                    const int col = n0 + cc, left = P.N - col;
                    if (left <= 0) break;  // the same for the whole warp
                    uint32_t r[16];
                    tmem_ld16(t0 + cc, r);
                    if (PAIR) {
                        uint32_t ru[16];
                        tmem_ld16(t0 + TN + cc, ru);
                        float bg[16], bu[16];
                        load_bias(P.bias ? P.bias + col : nullptr, left, bg);
                        load_bias(P.bias ? P.bias + P.F + col : nullptr, left, bu);
                        if (MODE == FWD) {
                            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                            float h[16];
                            if (P.act == 0) fwd16<T, 0>(r, ru, bg, bu, h);
                            else if (P.act == 1) fwd16<T, 1>(r, ru, bg, bu, h);
                            else if (P.act == 2) fwd16<T, 2>(r, ru, bg, bu, h);
                            else fwd16<T, 3>(r, ru, bg, bu, h);
                            if (row < P.M) store16((T*)P.out + (size_t)row * P.ldo + col, h, left, P.vec);
                        } else {
                            float dh[16], z[32];
                            if (row < P.M) load16((const T*)P.dh + (size_t)row * P.F + col, dh, left, P.vec);
                            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                            if (P.act == 0) dz16<T, 0>(r, ru, bg, bu, dh, z);
                            else if (P.act == 1) dz16<T, 1>(r, ru, bg, bu, dh, z);
                            else if (P.act == 2) dz16<T, 2>(r, ru, bg, bu, dh, z);
                            else dz16<T, 3>(r, ru, bg, bu, dh, z);
                            if (row < P.M) {
                                // z's rows are padded to whole 16-byte groups: always aligned
                                T* dst = (T*)P.out + (size_t)row * P.ldo + col;
                                store16(dst, z, left, true);
                                store16(dst + P.ldo / 2, z + 16, left, true);
                            }
                            if (P.db) {
                                if (row >= P.M) {  // rows behind the last one add nothing, whatever they hold
#pragma unroll
                                    for (int j = 0; j < 32; ++j) z[j] = 0.f;
                                }
                                const float s = column_sums(z, lane);
                                // one lane of one warp owns each of these sums: the additions keep their order
                                if ((lane & 15) < left)
                                    atomicAdd(P.db + ((size_t)blockIdx.x * 4 + q) * 2 * P.F + (lane < 16 ? 0 : P.F) + col + (lane & 15), s);
                            }
                        }
                    } else {
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                        if (row < P.M) {
                            float v[16];
#pragma unroll
                            for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[j]);
                            store16((T*)P.out + (size_t)row * P.ldo + col, v, left, P.vec);
                        }
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;");
                __syncwarp();
                if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(s32(&S.tempty[acc])) : "memory");
                if (++acc == 2) { acc = 0; accph ^= 1u; }
            }
        }
    }
    if (!ok) {
        S.stop = 1;
        atomicExch(&g_err, 1);
    }
    asm volatile("tcgen05.fence::before_thread_sync;");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;");
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * BN));
}

// dW from the partial tiles: tile t is the sum of the slots b + t of the CTAs whose shares of a block's units meet it,
// in the order of b.  One thread, 4 columns; grid: (rows of a tile) x tiles.
template <class T, int BN>
__global__ void __launch_bounds__(256) k_dw_sum(const float* part, T* dw, int F, int K, int tile0, int ntp, int blk, int ctas,
                                                int ntn) {
    constexpr int C4 = BN / 4;
    const int t = blockIdx.y, idx = blockIdx.x * 256 + threadIdx.x, r = idx / C4, c = (idx % C4) * 4;
    const int tile = tile0 + t, half_tiles = (F + BM - 1) / BM;
    const int mt = tile / ntn, up = mt >= half_tiles, f = (up ? mt - half_tiles : mt) * BM + r, k = (tile % ntn) * BN + c;
    if (f >= F || k >= K) return;
    const long long U = (long long)ntp * blk, lo = (long long)t * blk, hi = lo + blk;
    int b = (int)(lo * ctas / U);  // near the first CTA whose share ends behind lo
    while (b > 0 && U * b / ctas > lo) --b;
    while (U * (b + 1) / ctas <= lo) ++b;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (; b < ctas && U * b / ctas < hi; ++b) {
        if (U * (b + 1) / ctas == U * b / ctas) continue;  // an empty share
        const float4 v = __ldcs(reinterpret_cast<const float4*>(part + ((size_t)(b + t) * BM + r) * BN + c));
        s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    T* dst = dw + (size_t)(up ? F + f : f) * K + k;
    const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (k + j < K) {
            if constexpr (sizeof(T) == 4) dst[j] = v[j];
            else dst[j] = Half2<T>::one(v[j]);
        }
}

// db from the CTAs' column sums [rows][n]: 32 columns a block, 32 rows at a time, added in fp64
__global__ void __launch_bounds__(1024) k_db_sum(const float* part, float* db, int rows, int n) {
    __shared__ double sh[32][33];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5, col = blockIdx.x * 32 + x;
    double s = 0.0;
    if (col < n)
        for (int r = y; r < rows; r += 32) s += part[(size_t)r * n + col];
    sh[y][x] = s;
    __syncthreads();
    double v = sh[x][y];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (x == 0 && blockIdx.x * 32 + y < n) db[blockIdx.x * 32 + y] = (float)v;
}

// rows of 16-bit numbers copied to rows of `ldd` (a multiple of 8), zeros behind the n-th
__global__ void __launch_bounds__(256) k_pad(const uint16_t* src, long long ld, uint16_t* dst, int ldd, int n, long long rows) {
    const int groups = ldd / 8;
    const long long total = rows * groups;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long r = i / groups;
        const int c = (int)(i % groups) * 8;
        uint16_t v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = c + j < n ? src[r * ld + c + j] : (uint16_t)0;
        uint4 o;
        memcpy(&o, v, 16);
        *reinterpret_cast<uint4*>(dst + r * ldd + c) = o;
    }
}

// ------------------------------------------------------------------ host side
static bool map2d(CUtensorMap* m, int type, const void* base, long long cols, long long rows, long long ld, int box_rows) {
    EncodeTiledFn f = encode_fn();
    if (!f) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
    const cuuint32_t box[2] = {(cuuint32_t)BK, (cuuint32_t)box_rows};
    const cuuint32_t es[2] = {1, 1};
    return f(m, type == 1 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(base), dims,
             strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// the shared-memory limit is a property of (function, device)
template <class T, int MODE, int BN>
static cudaError_t launch(const Args& P, int grid, cudaStream_t st) {
    static std::once_flag once[64];
    static cudaError_t rc[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    std::call_once(once[dev], [dev]() {
        rc[dev] = cudaFuncSetAttribute(k_ff<T, MODE, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<BN>());
    });
    if (rc[dev] != cudaSuccess) return rc[dev];
    k_ff<T, MODE, BN><<<grid, NTH, smem_bytes<BN>(), st>>>(P);
    return cudaGetLastError();
}

static bool needs_pad(const void* p, long long ld, int cols) { return cols % 8 || ld % 8 || ((uintptr_t)p & 15); }
static long long up16(long long b) { return (b + 255) & ~255ll; }
static int pad8(int n) { return (n + 7) & ~7; }

struct Plan {
    long long xp, wp, z, db, part, total;  // offsets in the workspace
    bool padx, padw;
    int dw_bn, tiles, passes, ntp, ctas, blk;
};
// DW: passes of at most one tile a CTA (then a CTA's share meets two tiles at most)
static Plan plan(int M, int K, int F, const void* X, long long ldx, const void* W, int backward, int nsm) {
    Plan L = {};
    long long o = 0;
    L.padx = needs_pad(X, ldx, K);
    L.padw = needs_pad(W, K, K);
    auto take = [&](long long bytes) { const long long at = o; o += up16(bytes); return at; };
    L.xp = take(L.padx ? (long long)M * pad8(K) * 2 : 0);
    L.wp = take(L.padw ? 2ll * F * pad8(K) * 2 : 0);
    if (backward) {
        L.z = take((long long)M * 2 * pad8(F) * 2);
        L.db = take((long long)nsm * 4 * 2 * F * 4);
        L.dw_bn = K <= 128 ? 128 : 256;
        L.tiles = 2 * ((F + BM - 1) / BM) * ((K + L.dw_bn - 1) / L.dw_bn);
        L.passes = (L.tiles + nsm - 1) / nsm;
        L.ntp = (L.tiles + L.passes - 1) / L.passes;
        const int nk = (M + BK - 1) / BK;
        L.blk = nk < DW_BLOCK ? nk : DW_BLOCK;
        const long long units = (long long)L.ntp * L.blk;
        L.ctas = (int)(units < nsm ? units : nsm);
        L.part = take((long long)(L.ctas + L.ntp) * BM * L.dw_bn * 4);
    }
    L.total = o;
    return L;
}

static cudaError_t pad(const void* src, long long ld, void* dst, int cols, long long rows, cudaStream_t st) {
    const long long n = rows * (pad8(cols) / 8);
    const int grid = (int)std::min<long long>((n + 255) / 256, 148 * 16);
    k_pad<<<grid, 256, 0, st>>>((const uint16_t*)src, ld, (uint16_t*)dst, pad8(cols), cols, rows);
    return cudaGetLastError();
}

struct Call {
    int M, K, F, type, act;
    const void* X;
    long long ldx;
    const void* W;
    const float* b;
    uint8_t* ws;
    cudaStream_t st;
    int nsm;
};

static cudaError_t operands(Call& c, const Plan& L) {
    cudaError_t e = cudaSuccess;
    if (L.padx) {
        e = pad(c.X, c.ldx, c.ws + L.xp, c.K, c.M, c.st);
        c.X = c.ws + L.xp;
        c.ldx = pad8(c.K);
    }
    if (L.padw && e == cudaSuccess) {
        e = pad(c.W, c.K, c.ws + L.wp, c.K, 2ll * c.F, c.st);
        c.W = c.ws + L.wp;
    }
    return e;
}

template <class T>
static cudaError_t forward(Call c, const Plan& L, void* h) {
    cudaError_t e = operands(c, L);
    if (e != cudaSuccess) return e;
    const long long ldw = L.padw ? pad8(c.K) : c.K;
    Args P = {};
    if (!map2d(&P.a0, c.type, c.X, c.K, c.M, c.ldx, BM) || !map2d(&P.b0, c.type, c.W, c.K, c.F, ldw, 128) ||
        !map2d(&P.b1, c.type, (const T*)c.W + c.F * ldw, c.K, c.F, ldw, 128))
        return cudaErrorInvalidValue;
    P.M = c.M; P.N = c.F; P.F = c.F; P.act = c.act; P.bias = c.b;
    P.nk = (c.K + BK - 1) / BK;
    P.out = h; P.ldo = c.F;
    P.vec = c.F % 8 == 0 && ((uintptr_t)h & 15) == 0;
    const long long tiles = (long long)((c.M + BM - 1) / BM) * ((c.F + 127) / 128);
    return launch<T, FWD, 256>(P, (int)std::min<long long>(tiles, c.nsm), c.st);
}

template <class T, int BN>
static cudaError_t dw_passes(const Call& c, const Plan& L, Args P, void* dw, int dw_type) {
    const int ntn = (c.K + BN - 1) / BN;
    for (int t0 = 0; t0 < L.tiles; t0 += L.ntp) {
        P.tile0 = t0;
        P.ntp = std::min(L.ntp, L.tiles - t0);
        // as many CTAs as the full passes: a share never exceeds one tile
        const int ctas = (int)std::min<long long>((long long)P.ntp * L.blk, L.ctas);
        cudaError_t e = launch<T, DW, BN>(P, ctas, c.st);
        if (e != cudaSuccess) return e;
        const dim3 grid(BM * BN / 4 / 256, P.ntp);
        if (dw_type == 0) k_dw_sum<float, BN><<<grid, 256, 0, c.st>>>((const float*)P.out, (float*)dw, c.F, c.K, t0, P.ntp, L.blk, ctas, ntn);
        else k_dw_sum<T, BN><<<grid, 256, 0, c.st>>>((const float*)P.out, (T*)dw, c.F, c.K, t0, P.ntp, L.blk, ctas, ntn);
        e = cudaGetLastError();
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

template <class T>
static cudaError_t backward(Call c, const Plan& L, const void* dh, void* dx, void* dw, int dw_type, float* db) {
    cudaError_t e = operands(c, L);
    if (e != cudaSuccess) return e;
    const long long ldw = L.padw ? pad8(c.K) : c.K;
    const int Fp = pad8(c.F);
    T* z = (T*)(c.ws + L.z);
    const T* Wu = (const T*)c.W + c.F * ldw;
    {   // z = [dg | du] and the column sums
        Args P = {};
        if (!map2d(&P.a0, c.type, c.X, c.K, c.M, c.ldx, BM) || !map2d(&P.b0, c.type, c.W, c.K, c.F, ldw, 128) ||
            !map2d(&P.b1, c.type, Wu, c.K, c.F, ldw, 128))
            return cudaErrorInvalidValue;
        P.M = c.M; P.N = c.F; P.F = c.F; P.act = c.act; P.bias = c.b;
        P.nk = (c.K + BK - 1) / BK;
        P.out = z; P.ldo = 2 * Fp;
        P.dh = dh;
        P.vec = c.F % 8 == 0 && ((uintptr_t)dh & 15) == 0;
        const long long tiles = (long long)((c.M + BM - 1) / BM) * ((c.F + 127) / 128);
        const int grid = (int)std::min<long long>(tiles, c.nsm);
        if (db) {
            P.db = (float*)(c.ws + L.db);
            e = cudaMemsetAsync(P.db, 0, (size_t)grid * 4 * 2 * c.F * 4, c.st);
            if (e != cudaSuccess) return e;
        }
        e = launch<T, DZ, 256>(P, grid, c.st);
        if (e != cudaSuccess) return e;
        if (db) {
            k_db_sum<<<(2 * c.F + 31) / 32, 1024, 0, c.st>>>(P.db, db, grid * 4, 2 * c.F);
            e = cudaGetLastError();
            if (e != cudaSuccess) return e;
        }
    }
    if (dx) {
        Args P = {};
        if (!map2d(&P.a0, c.type, z, c.F, c.M, 2 * Fp, BM) || !map2d(&P.a1, c.type, z + Fp, c.F, c.M, 2 * Fp, BM) ||
            !map2d(&P.b0, c.type, c.W, c.K, c.F, ldw, BK) || !map2d(&P.b1, c.type, Wu, c.K, c.F, ldw, BK))
            return cudaErrorInvalidValue;
        P.M = c.M; P.N = c.K; P.F = c.F;
        P.nk = 2 * ((c.F + BK - 1) / BK);
        P.out = dx; P.ldo = c.K;
        P.vec = c.K % 8 == 0 && ((uintptr_t)dx & 15) == 0;
        const int bn = c.K <= 128 ? 128 : 256;
        const long long tiles = (long long)((c.M + BM - 1) / BM) * ((c.K + bn - 1) / bn);
        const int grid = (int)std::min<long long>(tiles, c.nsm);
        e = bn == 128 ? launch<T, DX, 128>(P, grid, c.st) : launch<T, DX, 256>(P, grid, c.st);
        if (e != cudaSuccess) return e;
    }
    if (dw) {
        Args P = {};
        if (!map2d(&P.a0, c.type, z, c.F, c.M, 2 * Fp, BK) || !map2d(&P.a1, c.type, z + Fp, c.F, c.M, 2 * Fp, BK) ||
            !map2d(&P.b0, c.type, c.X, c.K, c.M, c.ldx, BK))
            return cudaErrorInvalidValue;
        P.M = c.M; P.N = c.K; P.F = c.F;
        P.nk = (c.M + BK - 1) / BK;
        P.out = c.ws + L.part;
        e = L.dw_bn == 128 ? dw_passes<T, 128>(c, L, P, dw, dw_type) : dw_passes<T, 256>(c, L, P, dw, dw_type);
    }
    return e;
}

// tile indices are 32-bit
static bool shape_ok(int M, int K, int F) {
    return M >= 0 && K >= 1 && F >= 1 && M <= (1 << 30) && K <= (1 << 20) && F <= (1 << 20) &&
           ((long long)M / BM + 1) * ((long long)std::max(K, F) / 128 + 1) < (1ll << 30);
}

// shared argument checks; 0 when the call can run
static int check(const char* who, int M, int K, int F, int type, int act, const void* X, long long ldx, const void* W,
                 const float* b, const void* ws, long long ws_size, int backward, Plan* L, int* nsm) {
    auto bad = [&](const char* what) { set_error(-22, who, what); return -22; };
    if (!shape_ok(M, K, F)) return bad("invalid shape");
    if (type != 1 && type != 2) return bad("type must be 1 (bf16) or 2 (fp16)");
    if (act < 0 || act > 3) return bad("activation must be 0 tanh, 1 ELU, 2 SiLU or 3 GELU");
    if (ldx < K && M > 1) return bad("row stride below K");
    if (M > 0 && (!X || ((uintptr_t)X & 1))) return bad("null or misaligned X");
    if (!W || ((uintptr_t)W & 1) || ((uintptr_t)b & 3)) return bad("null or misaligned W or b");
    int dev = 0;
    *nsm = 148;
    cudaError_t e = cudaGetDevice(&dev);
    // the tensor maps are encoded by the driver, which needs the context current in this thread (autograd's own
    // threads come without)
    if (e == cudaSuccess) e = cudaSetDevice(dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(nsm, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) { set_error((int)e, who, cudaGetErrorString(e)); return -1; }
    *L = plan(M, K, F, X, ldx, W, backward, *nsm);
    if (L->total > 0 && (!ws || ((uintptr_t)ws & 255) || ws_size < L->total))
        return bad("workspace too small or not 256-byte aligned");
    return 0;
}

}  // namespace g1ff

extern "C" {

long long g1_gated_ff_workspace(int M, int K, int F, const void* X, long long ldx, const void* W, int backward) {
    if (!g1ff::shape_ok(M, K, F)) return 0;
    int dev = 0, nsm = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&nsm, cudaDevAttrMultiProcessorCount, dev);
    return g1ff::plan(M, K, F, X, ldx, W, backward, nsm).total;
}

int g1_gated_ff(int M, int K, int F, int type, int act, const void* X, long long ldx, const void* W, const float* b, void* h,
                void* ws, long long ws_size, void* stream) {
    g1ff::Plan L;
    g1ff::Call c = {M, K, F, type, act, X, M == 1 ? (long long)K : ldx, W, b, (uint8_t*)ws, (cudaStream_t)stream, 148};
    const int rc = g1ff::check("g1_gated_ff", M, K, F, type, act, X, c.ldx, W, b, ws, ws_size, 0, &L, &c.nsm);
    if (rc) return rc;
    if (M > 0 && (!h || ((uintptr_t)h & 1))) { set_error(-22, "g1_gated_ff", "null or misaligned h"); return -22; }
    if (M == 0) return 0;
    const cudaError_t e = type == 1 ? g1ff::forward<__nv_bfloat16>(c, L, h) : g1ff::forward<__half>(c, L, h);
    if (e != cudaSuccess) { set_error((int)e, "g1_gated_ff", cudaGetErrorString(e)); return -1; }
    return 0;
}

int g1_gated_ff_backward(int M, int K, int F, int type, int act, const void* dh, const void* X, long long ldx, const void* W,
                         const float* b, void* dx, void* dw, int dw_type, float* db, void* ws, long long ws_size,
                         void* stream) {
    g1ff::Plan L;
    g1ff::Call c = {M, K, F, type, act, X, M == 1 ? (long long)K : ldx, W, b, (uint8_t*)ws, (cudaStream_t)stream, 148};
    const int rc = g1ff::check("g1_gated_ff_backward", M, K, F, type, act, X, c.ldx, W, b, ws, ws_size, 1, &L, &c.nsm);
    if (rc) return rc;
    if ((dw_type != 0 && dw_type != type) || ((uintptr_t)dx & 1) || ((uintptr_t)dw & (dw_type == 0 ? 3 : 1)) ||
        ((uintptr_t)db & 3) || (M > 0 && (!dh || ((uintptr_t)dh & 1)))) {
        set_error(-22, "g1_gated_ff_backward", "dw must be fp32 or of the inputs' type; null or misaligned pointer");
        return -22;
    }
    cudaError_t e = cudaSuccess;
    if (M == 0) {  // sums over no rows
        if (dw) e = cudaMemsetAsync(dw, 0, 2 * (size_t)F * K * (dw_type == 0 ? 4 : 2), c.st);
        if (db && e == cudaSuccess) e = cudaMemsetAsync(db, 0, 2 * (size_t)F * 4, c.st);
    } else {
        e = type == 1 ? g1ff::backward<__nv_bfloat16>(c, L, dh, dx, dw, dw_type, db)
                      : g1ff::backward<__half>(c, L, dh, dx, dw, dw_type, db);
    }
    if (e != cudaSuccess) { set_error((int)e, "g1_gated_ff_backward", cudaGetErrorString(e)); return -1; }
    return 0;
}

int g1_gated_ff_status(void) {
    int v = 0, z = 0;
    if (cudaMemcpyFromSymbol(&v, g1ff::g_err, sizeof v) != cudaSuccess) return -1;
    if (v && cudaMemcpyToSymbol(g1ff::g_err, &z, sizeof z) != cudaSuccess) return -1;
    return v;
}

}  // extern "C"
