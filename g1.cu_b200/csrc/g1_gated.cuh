// g1_gated.cuh -- the gated feed-forward layer on the tensor cores (tcgen05), forward and backward:
//
//   g = X Wg^T + bg,  u = X Wu^T + bu,  h = act(g) * u          X [M][K], W [2F][K] = [Wg; Wu], b [2F]
//   dg = dh u act'(g),  du = dh act(g)
//   dX = dg Wg + du Wu,   dWg = dg^T X,  dWu = du^T X,   dbg = sum over rows of dg,  dbu = sum of du
//
// X, W, h and their gradients are bf16 or fp16, sums and everything between the products fp32; h, dX and dW are
// rounded once.  dg and du are rounded to the 16-bit type between the two backward products (they are
// operands of the tensor cores there).  That is as large an error of dX and dW as rounding the results, independent of it, and it
// does not average away, as the sums grow like their errors: 2.3e-3 of the norm in bf16 and 2.9e-4 in fp16, where rounding
// the results alone leaves 1.7e-3 and 2.1e-4; an fp32 dW has no rounding of its own but keeps this one, 1.7e-3 and 2.1e-4.  In
// fp16 dg and du overflow above 65504, and below 6e-5 they lose digits before dX and dW do: fp32 dW with dh of size 1e-4 is off by
// 3.1e-4, of size 1e-5 by 2.5e-3, so fp16 rows want a loss scale.  db is summed from the unrounded values.
//
// One kernel, k_ff, in several modes, all C = A B with fp32 accumulators in tensor memory, on 256 x 256 tiles by pairs of
// CTAs (cta_group::2: each CTA loads its 128 rows of A and half of B), or 128 x 128 / 64 by single ones where there
// are too few of those (tile_shape):
//
//   FWD  A = X, B = 128 rows of Wg and the same 128 rows of Wu, one MMA of N = 256; the epilogue holds g and u of
//        128 outputs side by side and writes h.  Neither g nor u leaves the SM.
//   DZ   the same product again; the epilogue reads dh and writes z = [dg | du] ([M][2 Fp]) and the column
//        sums.  Recomputing g and u costs 4MKF operations of the backward's 12MKF; keeping them at the accuracy
//        that db needs (fp32) would write and read 16 bytes an output, more time than the product up to K = 1024
//        or so, and hold 8 bytes an output between forward and backward.
//   DX   A = z, B = W read along its rows (MN-major): no transposed copy.
//   DW   A = z^T, B = X^T, both MN-major straight from their row-major tiles, summed over M.  The 2F x K tiles are
//        few and M is long: the work split stands at Tiles.  DXS: DX split the same way, for few rows and many outputs.
//   A few rows (up to ROWS_MAX) go forward by k_ff_rows, without tensor cores.
//
// Operands come by TMA (128-byte swizzle, zero fill past the edges, no multicast) in chunks of 64 along the sum, four to seven
// stages; one thread issues the loads, one the MMAs, up to sixteen warps run the epilogue of a tile while the
// next one accumulates in the other half of tensor memory.  Every wait is bounded; one that runs out sets a flag, an env's own
// (g1_env_tc_status) or the device's for all other calls (g1_gated_ff_status), and the kernel ends with garbage in its outputs.
//
// What bounds it: the products.  A chunk's 32 KB a CTA are written to and read from shared memory in the 512 cycles of its
// MMAs, close to the 128 bytes a cycle that it has (tensor pipe 74 % active in DX, 56 % in DZ, whose epilogue moves
// dh, dg and du through shared memory as well); under the power cap of a long step the clock gives way first.  Below
// K = 500 or so the epilogues do: 2.7 us a 128 x 128 tile and CTA in FWD, 4.2 us in DZ.
// Measured on one B200 (graph replays in short bursts; percent of the measured 1659 TFLOP/s):
//   forward 32768 x 1024 x 1024              98 us    1400 TFLOP/s   84 %; 116 us at length, at 1.40 GHz under the power cap
//   forward and backward 524288 x 1024 x 512 3.56 ms, 927 TFLOP/s of the 12MKF that cannot be avoided, 1236 of the 16MKF run;
//                                            4.2 ms at length, at 1.12 GHz.  FWD 0.80, DZ 0.93, DX 0.82, DW 0.84 each by itself
//   forward 65536 x 104 x 1024               73 us, its DZ 117 us by itself; 151 and 418 MB
//   forward 1 x 1024 x 1024                  2.5 us   1.7 TB/s from L2: latency
// Steps: 128-row tiles by single CTAs 117 us and 4.57 ms; pairs of CTAs 109 us and 4.29 ms; coalesced epilogue with
// two-number arithmetic 101 us and 3.9 ms; accumulators handed back before the stores, no bank conflicts 3.7 ms; DZ alone from
// 0.98 to 0.93 ms without spills (at K = 104 from 181 to 117 us).
// Taken out: the next tile's A fetched to L2 ahead, by the loading thread (115 us, 4.6 ms) or by the second CTA's idle MMA
// warp (no change); 8 epilogue warps of 64 columns (K = 104: 118 us, 16 warps 88).
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace g1ff {

using g1gemm::s32;

constexpr int BM = 128, BK = 64;  // rows of A a CTA, chunk of the sum
// DXS: DX with its sum cut, as DW's; DZU: DZ for rows of dh that do not start on 16-byte boundaries
enum { FWD = 0, DZ = 1, DX = 2, DW = 3, DXS = 4, DZU = 5 };
// CG: CTAs that work on a tile together (cta_group); BN: columns of B a tile
template <int MODE, int BN, int CG>
struct Cfg {
    static constexpr bool Z = MODE == DZ || MODE == DZU, PAIR = MODE == FWD || Z;
    static constexpr int TN = PAIR ? BN / 2 : BN;                  // output columns a tile
    static constexpr int PARTS = TN >= 64 ? 4 : TN / 16;           // epilogue warps a TMEM lane quarter
    static constexpr int EPI = 4 * PARTS, NTH = 64 + 32 * EPI;
    static constexpr int CW = TN / PARTS, SC = CW >= 32 ? 32 : 16; // columns a warp, and a step of it
    static constexpr int NB = BN / CG;                             // columns of B in this CTA's memory
    static constexpr int STAGES = Z ? 4 : MODE == FWD ? 5 : MODE == DX ? 6 : 7;
    // bytes of a warp's buffer: 32 rows x SC columns; DZ two of them and 32 x 16 more
    static constexpr int PIECE = 32 * SC * 2, AHEAD = MODE == DZ ? 2 : 1;
    static constexpr int BUF = MODE == DW || MODE == DXS ? 16 : AHEAD * PIECE + (Z ? 1024 : 0);
    static constexpr int STAGE_BYTES = (BM + NB) * BK * 2;
};
// The tensor cores truncate: each of the K/16 steps of a sum loses up to a step of fp32 of it, towards 0, so g and u come out
// smaller the longer the sum.  Of a sum whose terms come in no order a step finds half of it there on the average, and loses about
// half a step where its terms' bits reach below it: measured on normal x and w, K = 256 to 2048, 0.10 to 0.12 of 2^-23 of the result
// a step in bf16 and 0.14 in fp16.  DZ puts 1/8 back, as an fma in place of the addition of the bias: db at K = 1024 is off by 5.5e-7 of
// its norm instead of 1.1e-6, at K = 2048 by 1.2e-6 instead of 2.4e-6.  Sums whose largest terms come first lose twice as much, those
// whose largest come last a fifth (off by 14 instead of 2 of 2^-23 at K = 2048).  (FWD does not: it rounds h to 16 bits.)
constexpr float TRUNC = 1.f / (1 << 26);
constexpr int DW_BLOCK = 64;  // chunks (of 64 rows) that the CTAs of DW walk together

__device__ int g_err;    // a wait of a call that brings no flag of its own ran out
__device__ int g_taken;  // g_err as k_take_err found it

struct Args {
    CUtensorMap a0, a1, b0, b1;  // gate / up halves where they differ
    int M, N, nk;                // rows and columns of the output (FWD, DZ: N = F); chunks of the sum
    int F, act;
    const float* bias;           // [2F] or null
    const void* dh;              // DZ: [M][F]
    void* out;                   // h [M][F], z [M][2 Fp], dX [M][K], or the fp32 partial tiles
    long long ldo;
    float2 up;                   // DZ: what an accumulated g or u is multiplied by (see TRUNC)
    float* db;                   // DZ: [gridDim][4][2F] column sums, or null
    int tile0, ntp, blk;         // DW, DXS: the pass's tiles, chunks a block (see Tiles)
    int direct, out32;           // DW: every CTA has the whole sum of its tile: dW itself is written, in fp32 or 16 bits
    int vec;                     // rows of the output and of dh are 16-byte aligned
    int* err;                    // the flag of a wait that ran out; null: g_err
};

__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, uint32_t limit = g1gemm::SPIN) {
    const uint32_t a = s32(bar);
    for (uint32_t it = 0; it < limit; ++it) {
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

// for a whole warp: all lanes go on or none, as what follows (tcgen05.ld, ldmatrix) is for whole warps
__device__ __forceinline__ bool wait_all(uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)); }

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

// ---- two fp32 numbers an instruction
typedef unsigned long long f2;
__device__ __forceinline__ f2 mk(float x, float y) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ f2 mk(float2 v) { return mk(v.x, v.y); }
__device__ __forceinline__ f2 all(float x) { return mk(x, x); }
__device__ __forceinline__ float2 un(f2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ f2 add(f2 a, f2 b) {
    f2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f2 mul(f2 a, f2 b) {
    f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f2 fma(f2 a, f2 b, f2 c) {
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
// 2^x and 1/x of the special-function unit (2 and 1 units in the last place; results below 2^-126 are 0)
__device__ __forceinline__ f2 ex2(f2 v) {
    float2 x = un(v);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(x.x));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(x.y));
    return mk(x);
}
__device__ __forceinline__ f2 rcp(f2 v) {
    float2 x = un(v);
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(x.x));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(x.y));
    return mk(x);
}
constexpr float LOG2E = 1.4426950408889634f;

// act(g) and, with D, act'(g), in about 2^-21 of 1 + |g|; relative to act itself near 0 too.
//   tanh   1 - 2 / (1 + e^2|g|) with g's sign; its Taylor series to the 7th power where |g| < 0.2 (the rest is 6e-8 of g)
//   ELU    e^g - 1 below 0; its Taylor series to the 6th power where g > -0.25
//   SiLU   g s, s = 1 / (1 + e^-g); derivative s + g s (1 - s)
//   GELU   g Phi(g), derivative Phi(g) + g phi(g); with e = e^(-g^2 / 2) and t = 1 / (1 + p |g| / sqrt 2), Phi(-|g|) is e t P(t) / 2:
//          Abramowitz and Stegun, Handbook of Mathematical Functions, 7.1.26 (erf to 1.5e-7), the same e as phi's
// (CUDA's tanhf, expm1f and erff take 20 to 40 instructions a number, and the epilogue is what bounds DZ.)
template <int ACT, bool D>
__device__ __forceinline__ void act2(f2 g, f2& a, f2& d) {
    const f2 one = all(1.f);
    if (ACT == 0) {
        const float2 x = un(g);
        const f2 m = mk(fabsf(x.x), fabsf(x.y));
        const f2 r = rcp(add(ex2(mul(m, all(2.f * LOG2E))), one));
        const float2 big = un(fma(r, all(-2.f), one));
        const f2 q = mul(g, g);
        const float2 ser = un(mul(g, fma(q, fma(q, fma(q, all(-17.f / 315.f), all(2.f / 15.f)), all(-1.f / 3.f)), one)));
        a = mk(fabsf(x.x) < 0.2f ? ser.x : copysignf(big.x, x.x), fabsf(x.y) < 0.2f ? ser.y : copysignf(big.y, x.y));
        if (D) {
            // 1 - tanh^2 keeps its relative size as 4 r (1 - r)
            d = mul(mul(r, all(4.f)), fma(r, all(-1.f), one));
        }
    } else if (ACT == 1) {
        const float2 x = un(g);
        const f2 n = mk(x.x > 0.f ? 0.f : x.x, x.y > 0.f ? 0.f : x.y);  // keeps a NaN
        const float2 e = un(ex2(mul(n, all(LOG2E))));
        const float2 s = un(mul(
            n, fma(n, fma(n, fma(n, fma(n, fma(n, all(1.f / 720.f), all(1.f / 120.f)), all(1.f / 24.f)), all(1.f / 6.f)), all(0.5f)), one)));
        const float2 nn = un(n);
        a = mk(x.x > 0.f ? x.x : nn.x > -0.25f ? s.x : e.x - 1.f, x.y > 0.f ? x.y : nn.y > -0.25f ? s.y : e.y - 1.f);
        if (D) d = mk(e);
    } else if (ACT == 2) {
        const f2 s = rcp(add(ex2(mul(g, all(-LOG2E))), one));
        a = mul(g, s);
        if (D) d = fma(a, fma(s, all(-1.f), one), s);
    } else {
        const float2 x = un(g);
        const f2 m = mk(fabsf(x.x), fabsf(x.y));
        const f2 e = ex2(mul(mul(g, g), all(-0.5f * LOG2E)));
        const f2 t = rcp(fma(m, all(0.3275911f * 0.70710678118654752f), one));
        const f2 p = fma(t, fma(t, fma(t, fma(t, all(1.061405429f), all(-1.453152027f)), all(1.421413741f)), all(-0.284496736f)),
                         all(0.254829592f));
        const float2 c = un(mul(mul(e, all(0.5f)), mul(t, p)));  // Phi(-|g|)
        const f2 phi = mk(x.x > 0.f ? 1.f - c.x : c.x, x.y > 0.f ? 1.f - c.y : c.y);
        a = mul(g, phi);
        if (D) d = fma(mul(g, all(0.39894228040143268f)), e, phi);
    }
}

// 16 TMEM lanes x 16 columns: lane l holds columns 2 (l % 4), + 1 and 8 further on of rows l / 4 and l / 4 + 8, as
// r[4 k + 2 i + c] = (row l / 4 + 8 i, column 8 k + 2 (l % 4) + c)
__device__ __forceinline__ void tmem_ld16x16(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

// A launch may start while the one before it in the stream ends (programmatic dependent launch): set up, then wait here
// before the first access to memory that another kernel writes.  The kernel is resident while that one still writes, so it
// reads by ordinary loads: read-only ones (ld.global.nc, which the compiler also makes of const __restrict__ arguments) want
// their data to stay as it is for as long as the kernel lives.
__device__ __forceinline__ void after_previous() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
}

template <int MODE, int BN, int CG>
struct Smem {
    using C = Cfg<MODE, BN, CG>;
    uint8_t a[C::STAGES][BM * BK * 2];
    uint8_t b[C::STAGES][C::NB * BK * 2];
    uint8_t buf[C::BUF > 16 ? C::EPI : 1][C::BUF];
    float bias[C::PAIR ? C::EPI : 1][C::AHEAD][2][32];
    uint64_t full[C::STAGES], empty[C::STAGES], tfull[2], tempty[2];
    uint32_t tslot;
    volatile int stop;  // a wait of this CTA ran out
};
template <int MODE, int BN, int CG>
constexpr int smem_bytes() { return (int)sizeof(Smem<MODE, BN, CG>) + 1024; }

// A warp's 32 rows x SC columns go to and from global memory through its buffer, so that neighbouring lanes touch
// neighbouring addresses (one row a lane would touch 32 lines with each access).  In the buffer the 16-byte groups of a
// row are permuted so that a column group over 8 rows, and neighbouring groups, lie in different banks.
// (8 rows further down the permutation is the same: an address moves on by a constant.)
template <int SC>
__device__ __forceinline__ int at(int r, int group) {
    return SC == 32 ? r * 64 + ((group ^ ((r >> 1) & 3)) << 4) : r * 32 + ((group ^ ((r >> 2) & 1)) << 4);
}
// to rows of m; vec: they start on 16-byte boundaries
template <class T, int SC>
__device__ __forceinline__ void rows_out(const uint8_t* buf, T* m, long long ld, int row0, int M, int col, int N, bool vec,
                                         int lane) {
    if (vec) {
        constexpr int CH = SC / 8, RS = 32 / CH;
        const int ch = lane % CH, r = lane / CH;
        T* dst = m + (size_t)(row0 + r) * ld + col + 8 * ch;
        const uint8_t* src = buf + at<SC>(r, ch);
        const bool inside = col + 8 * ch < N;
        if (row0 + 32 <= M && col + SC <= N) {  // the whole piece
#pragma unroll
            for (int i = 0; i < CH; ++i, dst += RS * ld)
                *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src + i * RS * SC * 2);
        } else {
#pragma unroll
            for (int i = 0; i < CH; ++i, dst += RS * ld)
                if (row0 + r + i * RS < M && inside)
                    *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src + i * RS * SC * 2);
        }
    } else {
        const int c = lane % SC;
#pragma unroll 8
        for (int i = 0; i < SC; ++i) {
            const int r = lane / SC + i * (32 / SC);
            if (row0 + r < M && col + c < N)
                m[(size_t)(row0 + r) * ld + col + c] = *reinterpret_cast<const T*>(buf + at<SC>(r, c / 8) + c % 8 * 2);
        }
    }
}

// v[0..3] summed over the 8 lanes of equal l % 4: halves of the list change sides twice; lane l gets the sum of
// v[2 (l / 16) + (l / 8) % 2]
__device__ __forceinline__ float sums4(const float* v, int lane) {
    const bool hi = lane & 16, mid = lane & 8;
    float a = hi ? v[2] : v[0], b = hi ? v[3] : v[1];
    a += __shfl_xor_sync(0xffffffffu, hi ? v[0] : v[2], 16);
    b += __shfl_xor_sync(0xffffffffu, hi ? v[1] : v[3], 16);
    const float s = (mid ? b : a) + __shfl_xor_sync(0xffffffffu, mid ? a : b, 8);
    return s + __shfl_xor_sync(0xffffffffu, s, 4);
}

__device__ __forceinline__ f2 acc2(const uint32_t* r) { return mk(__uint_as_float(r[0]), __uint_as_float(r[1])); }

// h of 8 columns of a row
template <int ACT>
__device__ __forceinline__ void fwd8(const uint32_t* rg, const uint32_t* ru, const float* bg, const float* bu, float* h) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        f2 a, d;
        act2<ACT, false>(add(acc2(rg + j), mk(bg[j], bg[j + 1])), a, d);
        *reinterpret_cast<float2*>(h + j) = un(mul(a, add(acc2(ru + j), mk(bu[j], bu[j + 1]))));
    }
}
// 32 rows x 8 columns of 16-bit numbers as four 8 x 8 matrices: lane l gives the address of row l and holds
// w[i] = (row 8 i + l / 4, columns 2 (l % 4), + 1)
__device__ __forceinline__ void load_rows(uint32_t addr, uint32_t* w) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void store_rows(uint32_t addr, const uint32_t* w) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                 : "memory");
}

// 16 or 4 bytes to shared memory behind the threads' back, zeros where ok is false
__device__ __forceinline__ void fetch16(uint32_t dst, const void* src, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void fetch4(uint32_t dst, const void* src, bool ok) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(ok ? 4 : 0) : "memory");
}

// z of 32 rows x 16 columns, the s0-th on: dh in `buf` is replaced by dg, du goes to `buf2` (16 columns); the column
// sums over the rows to sum[k][]: columns 8 k + 2 (l % 4), + 1 of dg, then of du
template <class T, int ACT, int SC>
__device__ __forceinline__ void dz16(const uint32_t (&rg)[2][8], const uint32_t (&ru)[2][8], const float (*sb)[32], const float2& up, int s0,
                                     uint32_t buf, uint32_t buf2, float (&sum)[2][4], int lane) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int c = s0 + 8 * k + 2 * (lane & 3);
        const f2 bg = *reinterpret_cast<const f2*>(&sb[0][c]), bu = *reinterpret_cast<const f2*>(&sb[1][c]);
        f2 sg = 0, su = 0;
        const uint32_t place = buf + at<SC>(lane, s0 / 8 + k);
        uint32_t w[4], v[4];
        load_rows(place, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f2 dh = mk(Half2<T>::unpack(w[i]));
            f2 a, d;
            act2<ACT, true>(fma(acc2(&rg[i / 2][4 * k + 2 * (i & 1)]), mk(up), bg), a, d);
            const f2 dg = mul(mul(dh, fma(acc2(&ru[i / 2][4 * k + 2 * (i & 1)]), mk(up), bu)), d), du = mul(dh, a);
            const float2 x = un(dg), y = un(du);
            w[i] = Half2<T>::pack(x.x, x.y);
            v[i] = Half2<T>::pack(y.x, y.y);
            sg = add(sg, dg);
            su = add(su, du);
        }
        store_rows(place, w);
        store_rows(buf2 + at<16>(lane, k), v);
        const float2 x = un(sg), y = un(su);
        sum[k][0] = x.x; sum[k][1] = x.y; sum[k][2] = y.x; sum[k][3] = y.y;
    }
}
template <class T>
__device__ __forceinline__ uint4 pack8(const float* v) {
    return make_uint4(Half2<T>::pack(v[0], v[1]), Half2<T>::pack(v[2], v[3]), Half2<T>::pack(v[4], v[5]),
                      Half2<T>::pack(v[6], v[7]));
}

// 16 neighbours of a row of dW, `n` of them inside it
template <class T>
__device__ __forceinline__ void store16(T* dst, const float* v, int n, bool vec) {
    if (vec && n >= 16) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < 4; ++j) reinterpret_cast<float4*>(dst)[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        } else {
            reinterpret_cast<uint4*>(dst)[0] = pack8<T>(v);
            reinterpret_cast<uint4*>(dst)[1] = pack8<T>(v + 8);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (j < n) {
                if constexpr (sizeof(T) == 4) dst[j] = v[j];
                else dst[j] = Half2<T>::one(v[j]);
            }
    }
}

// ---- two CTAs on a tile
__device__ __forceinline__ uint32_t cta_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t at_leader(uint32_t saddr) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(saddr));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
// a load into this CTA's memory; its bytes count at `bar`, which may lie in the tile's first CTA
template <int CG>
__device__ __forceinline__ void load2d(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    if constexpr (CG == 1)
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
                s32(dst)),
            "l"(map), "r"(x), "r"(y), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], "
            "[%4];" ::"r"(s32(dst)),
            "l"(map), "r"(x), "r"(y), "r"(bar)
            : "memory");
}
template <int CG>
__device__ __forceinline__ void mma16(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t accum) {
    if constexpr (CG == 1)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(ad), "l"(bd), "r"(idesc), "r"(accum));
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(ad), "l"(bd), "r"(idesc), "r"(accum));
}
// arrives on the barrier at this offset in every CTA of the tile once the MMAs issued so far are done
template <int CG>
__device__ __forceinline__ void commit(uint64_t* bar) {
    if constexpr (CG == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(s32(bar)) : "memory");
    else
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(s32(bar)),
            "h"((uint16_t)3)
            : "memory");
}

// The tiles of a CTA (of a group of CG).  FWD, DZ, DX: row blocks by column tiles, columns fastest, so that the CTAs in flight
// share rows of A in L2 and A comes from HBM once (the weights stay in L2).
// DW: the sum over M is cut for the CTAs to be equally loaded, each CTA keeping at most two tiles (two
// accumulators) from start to end: rows are walked in blocks of DW_BLOCK chunks, and of each block's ntp x DW_BLOCK
// (tile, chunk) units CTA b takes the same b-th share.  All CTAs stay within a block of rows, so X and z come from HBM
// once; cutting each tile's whole M into runs instead would have the tiles read the same rows at different times.
template <int MODE>
struct Tiles {
    int tile, step;                  // FWD, DZ, DX: this CTA's first tile, the distance to its next
    int t0, c0, c1, c2, blk;         // DW, DXS: chunks [c0, c1) of tile t0 and [0, c2) of tile t0 + 1 in each block
    // id-th of n CTAs (or groups of CTAs)
    __device__ __forceinline__ Tiles(const Args& P, int id, int n) {
        if (MODE == DW || MODE == DXS) {
            blk = P.blk;
            const long long U = (long long)P.ntp * blk;
            const long long u0 = U * id / n, u1 = U * (id + 1) / n;
            t0 = (int)(u0 / blk);
            c0 = (int)(u0 % blk);
            c1 = (int)min((long long)blk, c0 + (u1 - u0));
            c2 = (int)(u1 - u0) - (c1 - c0);
        } else {
            tile = id;
            step = n;
        }
    }
};

// a tile's place, moved on without a division
struct Place {
    int m, n, dm, dn, ntn;
    __device__ __forceinline__ Place(int tile, int step, int ntn_) : m(tile / ntn_), n(tile % ntn_), dm(step / ntn_), dn(step % ntn_), ntn(ntn_) {}
    __device__ __forceinline__ void next() {
        m += dm;
        n += dn;
        if (n >= ntn) { n -= ntn; ++m; }
    }
};

template <class T, int MODE, int BN, int CG>
__global__ void __launch_bounds__((Cfg<MODE, BN, CG>::NTH), 1) k_ff(const __grid_constant__ Args P) {
    using C = Cfg<MODE, BN, CG>;
    extern __shared__ uint8_t smem_raw[];
    auto& S = *reinterpret_cast<Smem<MODE, BN, CG>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    constexpr bool A_MN = MODE == DW, PAIR = C::PAIR, Z = C::Z, B_MN = !PAIR, CUT = MODE == DW || MODE == DXS;
    constexpr int TN = C::TN, STAGES = C::STAGES, NB = C::NB;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = CG == 1 ? 0 : (int)cta_rank();
    const int ntn = (P.N + TN - 1) / TN;
    // DW: 128-row tiles of the gate half, then of the up half
    const int half_tiles = (P.F + BM - 1) / BM;
    const int ntm = MODE == DW ? 2 * half_tiles / CG : (P.M + BM * CG - 1) / (BM * CG);
    const int ntiles = ntm * ntn, nk = P.nk;
    if (tid == 32) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&P.a0) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&P.b0) : "memory");
    }
    if (tid == 0) {
        S.stop = 0;
        for (int i = 0; i < STAGES; ++i) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(s32(&S.full[i])));
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(s32(&S.empty[i])));
        }
        for (int i = 0; i < 2; ++i) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(s32(&S.tfull[i])));
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(s32(&S.tempty[i])), "r"(CG * C::EPI));
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        __syncwarp();
        if constexpr (CG == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(&S.tslot)), "r"(2 * BN));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        } else {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(&S.tslot)), "r"(2 * BN));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;");
    __syncthreads();
    if (CG > 1) cluster_sync();  // the other CTA's barriers are ready
    asm volatile("tcgen05.fence::after_thread_sync;");
    const uint32_t tmem = S.tslot;
    bool ok = true;
    after_previous();
    const Tiles<MODE> W(P, blockIdx.x / CG, gridDim.x / CG);

    if (warp == 0 && lane == 0) {  // loads: this CTA's rows of A and its share of B
        int stage = 0;
        uint32_t phase = 0;
        auto load = [&](int tile, int c) -> bool {
            if (!wait(&S.empty[stage], phase ^ 1u)) return false;
            uint32_t bar = s32(&S.full[stage]);
            if (rank == 0)
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(CG * C::STAGE_BYTES)
                             : "memory");
            if (CG > 1) bar = at_leader(bar);
            const int mt = (tile / ntn) * CG + rank, n0 = (tile % ntn) * TN;
            uint8_t *as = S.a[stage], *bs = S.b[stage];
            if (PAIR) {
                load2d<CG>(as, &P.a0, c * BK, mt * BM, bar);
                if (CG == 1) {
                    load2d<CG>(bs, &P.b0, c * BK, n0, bar);
                    load2d<CG>(bs + TN * BK * 2, &P.b1, c * BK, n0, bar);
                } else {
                    load2d<CG>(bs, rank == 0 ? &P.b0 : &P.b1, c * BK, n0, bar);
                }
            } else if (MODE == DX || MODE == DXS) {
                // the sum runs over the gate half's columns, then the up half's
                const bool up = c >= nk / 2;
                const int k0 = (up ? c - nk / 2 : c) * BK;
                load2d<CG>(as, up ? &P.a1 : &P.a0, k0, mt * BM, bar);
#pragma unroll
                for (int j = 0; j < NB / 64; ++j)
                    load2d<CG>(bs + j * 8192, up ? &P.b1 : &P.b0, n0 + rank * NB + 64 * j, k0, bar);
            } else {
                const bool up = mt >= half_tiles;
                const int f0 = (up ? mt - half_tiles : mt) * BM;
#pragma unroll
                for (int j = 0; j < BM / 64; ++j) load2d<CG>(as + j * 8192, up ? &P.a1 : &P.a0, f0 + 64 * j, c * BK, bar);
#pragma unroll
                for (int j = 0; j < NB / 64; ++j) load2d<CG>(bs + j * 8192, &P.b0, n0 + rank * NB + 64 * j, c * BK, bar);
            }
            if (++stage == STAGES) { stage = 0; phase ^= 1u; }
            return true;
        };
        if (CUT) {
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
        // every load of this CTA has landed before it leaves: the first CTA's MMA thread has seen them all, or gave up
    } else if (warp == 1 && lane == 0 && rank == 0) {  // MMAs, of both CTAs
        constexpr uint32_t idesc = (1u << 4) | (Half2<T>::fmt << 7) | (Half2<T>::fmt << 10) | ((A_MN ? 1u : 0u) << 15) |
                                   ((B_MN ? 1u : 0u) << 16) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(CG * BM >> 4) << 24);
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
                mma16<CG>(d, ad, bd, idesc, (!first || k > 0) ? 1u : 0u);
            }
            commit<CG>(&S.empty[stage]);
            if (++stage == STAGES) { stage = 0; phase ^= 1u; }
            return true;
        };
        if (CUT) {
            for (int base = 0; base < nk && ok; base += W.blk) {
                for (int c = W.c0; c < W.c1 && ok; ++c)
                    if (base + c < nk) ok = mma(tmem, base == 0 && c == W.c0);
                for (int c = 0; c < W.c2 && ok; ++c)
                    if (base + c < nk) ok = mma(tmem + BN, base == 0 && c == 0);
            }
            if (ok) { commit<CG>(&S.tfull[0]); commit<CG>(&S.tfull[1]); }
        } else {
            uint32_t acc = 0, accph = 0;
            for (int tile = W.tile; tile < ntiles && ok; tile += W.step) {
                if (!wait(&S.tempty[acc], accph ^ 1u)) { ok = false; break; }
                asm volatile("tcgen05.fence::after_thread_sync;");
                for (int c = 0; c < nk && ok; ++c) ok = mma(tmem + acc * BN, c == 0);
                if (ok) commit<CG>(&S.tfull[acc]);
                if (++acc == 2) { acc = 0; accph ^= 1u; }
            }
        }
    } else if (warp >= 2) {  // epilogue: warp w reads TMEM lanes 32 (w & 3) .., part (w - 2) / 4 of the columns
        const int q = warp & 3, part = (warp - 2) >> 2;
        constexpr int CW = C::CW, SC = C::SC;
        const uint32_t tl = tmem + ((uint32_t)(32 * q) << 16);
        if (CUT) {
            // fp32 partial tiles, row-major; slot (group + tile) is this group's alone (the next share raises one of them)
            for (int a = 0; a < 2 && ok; ++a) {
                const bool have = a == 0 ? W.c1 > W.c0 : W.c2 > 0;
                if (!have) continue;
                // all of the CTA's products lie before this: as long as 64 other waits, or until one of those ran out
                ok = false;
                for (int i = 0; i < 64 && !ok && !__any_sync(0xffffffffu, S.stop); ++i) ok = wait_all(&S.tfull[a], 0);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;");
                const size_t row = ((size_t)(blockIdx.x / CG + W.t0 + a) * CG + rank) * BM + 32 * q + lane;
                float* dst = (float*)P.out + row * BN + part * CW;
                const int tile = P.tile0 + W.t0 + a, mt = (tile / ntn) * CG + rank, up = mt >= half_tiles;
                const int f = (up ? mt - half_tiles : mt) * BM + 32 * q + lane, k0 = (tile % ntn) * TN + part * CW;
#pragma unroll 1
                for (int cc = 0; cc < CW; cc += 16) {
                    uint32_t r[16];
                    tmem_ld16(tl + a * BN + part * CW + cc, r);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    if (MODE == DW && P.direct) {
                        if (f < P.F) {
                            float v[16];
#pragma unroll
                            for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[j]);
                            const size_t at0 = (size_t)(up ? P.F + f : f) * P.N + k0 + cc;
                            if (P.out32) store16((float*)P.out + at0, v, P.N - k0 - cc, P.vec);
                            else store16((T*)P.out + at0, v, P.N - k0 - cc, P.vec);
                        }
                        __syncwarp();  // the next columns are read by whole warps
                        continue;
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        reinterpret_cast<uint4*>(dst + cc)[j] = make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
                }
            }
        } else {
            uint32_t acc = 0, accph = 0;
            constexpr int CH = SC / 8, RS = 32 / CH, AHEAD = C::AHEAD;  // 16-byte groups a row, rows a step of rows_out
            uint8_t* buf = S.buf[warp - 2];
            float(*bias)[2][32] = S.bias[PAIR ? warp - 2 : 0];
            // Z: column (counted from a 16-column step's first) that this lane's sums are of, in its 8-column half
            const int mycol = 2 * (lane & 3) + ((lane >> 3) & 1);
            float* mydb = Z && P.db && !(lane & 4) ? P.db + ((size_t)blockIdx.x * 4 + q) * 2 * P.F + (lane & 16 ? P.F : 0) : nullptr;
            if (Z && mydb) {
                // the sums start at 0; the additions below are the same thread's, so they come after
                for (int c = part * CW + mycol; c < P.N; c += TN)
                    for (int e = 0; e < CW; e += 8)
                        if (c + e < P.N) mydb[c + e] = 0.f;
            }
            // The bias (a column a lane) and dh of a step are asked for one step ahead, a tile's first before the wait for its
            // products: in DZ by asynchronous copies into the other of two buffers, else through registers (which DZ has
            // none to spare of: with dh in them it spilled, 171 us instead of 117 at 65536 x 104 x 1024).
            uint32_t nx[MODE == DZU ? SC / 2 : 1];
            float nbg = 0.f, nbu = 0.f;
            auto ask = [&](const Place& to, int cc, int into) {
                if (!PAIR || to.m >= ntm) return;
                const int col = to.n * TN + part * CW + cc, row0 = (to.m * CG + rank) * BM + 32 * q;
                const bool b = P.bias && lane < SC && col + lane < P.N;
                const float* bg = P.bias + col + lane;
                if (MODE == DZ) {
                    if (lane < SC) {
                        fetch4(s32(&bias[into][0][lane]), b ? (const void*)bg : P.dh, b);
                        fetch4(s32(&bias[into][1][lane]), b ? (const void*)(bg + P.F) : P.dh, b);
                    }
                    const int ch = lane % CH, r = row0 + lane / CH;
                    const T* src = (const T*)P.dh + (size_t)r * P.F + col + 8 * ch;
                    const uint32_t dst = s32(buf) + into * C::PIECE + at<SC>(lane / CH, ch);
#pragma unroll
                    for (int i = 0; i < CH; ++i, src += (size_t)RS * P.F) {
                        const bool ok = r + i * RS < P.M && col + 8 * ch < P.N;
                        fetch16(dst + i * RS * SC * 2, ok ? (const void*)src : P.dh, ok);
                    }
                } else {
                    nbg = b ? *bg : 0.f;
                    nbu = b ? bg[P.F] : 0.f;
                }
                if (MODE == DZU) {  // one number a lane and access, two packed
                    const uint16_t* d16 = reinterpret_cast<const uint16_t*>(P.dh);
                    const int c = col + lane % SC;
#pragma unroll
                    for (int i = 0; i < SC; ++i) {
                        const int r = row0 + lane / SC + i * (32 / SC);
                        const uint32_t x = r < P.M && c < P.N ? d16[(size_t)r * P.F + c] : 0;
                        nx[MODE == DZU ? i / 2 : 0] = i & 1 ? nx[MODE == DZU ? i / 2 : 0] | (x << 16) : x;
                    }
                }
            };
            Place here(W.tile, W.step, ntn);
            int cur = 0;
            ask(here, 0, 0);
            for (int tile = W.tile; tile < ntiles; tile += W.step) {
                if (!wait_all(&S.tfull[acc], accph)) { ok = false; break; }
                asm volatile("tcgen05.fence::after_thread_sync;");
                const int row0 = (here.m * CG + rank) * BM + 32 * q, col0 = here.n * TN + part * CW;
                const uint32_t t0 = tl + acc * BN + part * CW;
                // hands the accumulator back once this warp has read its last columns of it.  Nothing but those reads has
                // to be over by then: a release at cluster scope would wait for the rows written before as well (22 % of
                // the epilogue's time at K = 104)
                bool held = true;
                auto release = [&]() {
                    asm volatile("tcgen05.fence::before_thread_sync;");
                    __syncwarp();
                    if (lane == 0) {
                        if (CG == 1)
                            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(s32(&S.tempty[acc])) : "memory");
                        else
                            asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(at_leader(s32(&S.tempty[acc])))
                                         : "memory");
                    }
                    held = false;
                };
#pragma unroll 1
                for (int cc = 0; cc < CW; cc += SC) {
                    const int col = col0 + cc;
                    const bool some = col < P.N;  // the same for the whole warp
                    if (MODE == DZ) asm volatile("cp.async.wait_all;" ::: "memory");
                    if (MODE != DZ && PAIR && some) {
                        if (lane < SC) { bias[0][0][lane] = nbg; bias[0][1][lane] = nbu; }
                        if (MODE == DZU) {
#pragma unroll
                            for (int i = 0; i < SC; ++i)
                                *reinterpret_cast<uint16_t*>(buf + at<SC>(lane / SC + i * (32 / SC), lane % SC / 8) + lane % 8 * 2) =
                                    (uint16_t)(nx[MODE == DZU ? i / 2 : 0] >> (16 * (i & 1)));
                        }
                    }
                    __syncwarp();
                    if (cc + SC < CW) {
                        ask(here, cc + SC, cur ^ 1);
                    } else {
                        Place then = here;
                        then.next();
                        ask(then, 0, cur ^ 1);
                    }
                    uint8_t* mine = buf + (AHEAD == 2 ? cur * C::PIECE : 0);
                    const float(*sb)[32] = bias[AHEAD == 2 ? cur : 0];
                    cur ^= 1;
                    if (!some) continue;
#pragma unroll 1
                    for (int s = 0; s < SC; s += 16) {
                        if (Z) {
                            uint8_t* du = buf + AHEAD * C::PIECE;
                            uint32_t rg[2][8], ru[2][8];
                            tmem_ld16x16(t0 + cc + s, rg[0]);
                            tmem_ld16x16(t0 + (16u << 16) + cc + s, rg[1]);
                            tmem_ld16x16(t0 + TN + cc + s, ru[0]);
                            tmem_ld16x16(t0 + (16u << 16) + TN + cc + s, ru[1]);
                            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                            if (cc + s + 16 == CW) release();
                            float sum[2][4];
                            if (P.act == 0) dz16<T, 0, SC>(rg, ru, sb, P.up, s, s32(mine), s32(du), sum, lane);
                            else if (P.act == 1) dz16<T, 1, SC>(rg, ru, sb, P.up, s, s32(mine), s32(du), sum, lane);
                            else if (P.act == 2) dz16<T, 2, SC>(rg, ru, sb, P.up, s, s32(mine), s32(du), sum, lane);
                            else dz16<T, 3, SC>(rg, ru, sb, P.up, s, s32(mine), s32(du), sum, lane);
                            if (P.db) {  // rows behind the last one have dh = 0
#pragma unroll
                                for (int k = 0; k < 2; ++k) {
                                    const float v = sums4(sum[k], lane);
                                    // one lane of one warp owns each of these sums: the additions keep their order
                                    const int c = col + s + 8 * k + mycol;
                                    if (mydb && c < P.N) atomicAdd(mydb + c, v);
                                }
                            }
                            __syncwarp();
                            // z's rows are padded to whole 16-byte groups
                            rows_out<T, 16>(du, (T*)P.out + P.ldo / 2, P.ldo, row0, P.M, col + s, P.N, true, lane);
                            __syncwarp();
                            continue;
                        }
                        uint32_t r[16];
                        tmem_ld16(t0 + cc + s, r);
                        uint32_t ru[16];
                        if (MODE == FWD) tmem_ld16(t0 + TN + cc + s, ru);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                        if (cc + s + 16 == CW) release();
#pragma unroll
                        for (int e = 0; e < 16; e += 8) {
                            float h[8];
                            if (MODE == FWD) {
                                float bg[8], bu[8];
                                *reinterpret_cast<float4*>(bg) = *reinterpret_cast<const float4*>(&sb[0][s + e]);
                                *reinterpret_cast<float4*>(bg + 4) = *reinterpret_cast<const float4*>(&sb[0][s + e + 4]);
                                *reinterpret_cast<float4*>(bu) = *reinterpret_cast<const float4*>(&sb[1][s + e]);
                                *reinterpret_cast<float4*>(bu + 4) = *reinterpret_cast<const float4*>(&sb[1][s + e + 4]);
                                if (P.act == 0) fwd8<0>(r + e, ru + e, bg, bu, h);
                                else if (P.act == 1) fwd8<1>(r + e, ru + e, bg, bu, h);
                                else if (P.act == 2) fwd8<2>(r + e, ru + e, bg, bu, h);
                                else fwd8<3>(r + e, ru + e, bg, bu, h);
                            } else {
#pragma unroll
                                for (int j = 0; j < 8; ++j) h[j] = __uint_as_float(r[e + j]);
                            }
                            *reinterpret_cast<uint4*>(mine + at<SC>(lane, (s + e) / 8)) = pack8<T>(h);
                        }
                    }
                    __syncwarp();
                    rows_out<T, SC>(mine, (T*)P.out, P.ldo, row0, P.M, col, P.N, Z || P.vec, lane);
                    __syncwarp();
                }
                if (held) release();  // columns behind the last one
                here.next();
                if (++acc == 2) { acc = 0; accph ^= 1u; }
            }
            if (MODE == DZ) asm volatile("cp.async.wait_all;" ::: "memory");  // nothing in flight, even after a wait that ran out
        }
    }
    if (!ok) {
        S.stop = 1;
        atomicExch(P.err ? P.err : &g_err, 1);
        if (warp == 0)  // give loads in flight 0.1 s to land
            for (int i = 0; i < 100; ++i) __nanosleep(1000000);
    }
    asm volatile("tcgen05.fence::before_thread_sync;");
    __syncthreads();
    if (CG > 1) cluster_sync();  // neither CTA leaves while the other reads its memory or arrives on its barriers
    asm volatile("tcgen05.fence::after_thread_sync;");
    if (warp == 0) {
        __syncwarp();
        if constexpr (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * BN));
        else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * BN));
    }
}

// db from the CTAs' column sums [rows][n]: 8 columns a block of 256 threads, 32 rows at a time, added in fp64
__device__ __forceinline__ void db_sum(const float* part, float* db, int rows, int n, int block) {
    const int x = threadIdx.x & 7, y = threadIdx.x >> 3, col = block * 8 + x;
    __shared__ double sh[32][9];
    double s = 0.0;
    if (col < n)
#pragma unroll 8
        for (int r = y; r < rows; r += 32) s += part[(size_t)r * n + col];
    sh[y][x] = s;
    __syncthreads();
    if (threadIdx.x < 8 && col < n) {
        double v = 0.0;
        for (int i = 0; i < 32; ++i) v += sh[i][x];
        db[col] = (float)v;
    }
}

// dW from the partial tiles: tile t is the sum of the slots b + t of the groups of CTAs whose shares of a block's units meet
// it, in the order of b.  One thread, 4 columns; grid: (rows of a tile) x tiles.  Further blocks (blockIdx.y >= ntp)
// sum db.
template <class T, int BN, int CG>
__global__ void __launch_bounds__(256) k_dw_sum(const float* part, T* dw, int F, int K, int tile0, int ntp, int blk, int groups,
                                                int ntn, const float* db_part, float* db, int db_rows) {
    constexpr int C4 = BN / 4, R = BM * CG;
    const int t = blockIdx.y;
    if (t >= ntp) {
        after_previous();
        db_sum(db_part, db, db_rows, 2 * F, (t - ntp) * gridDim.x + blockIdx.x);
        return;
    }
    const int idx = blockIdx.x * 256 + threadIdx.x, r = idx / C4, c = (idx % C4) * 4;
    const int tile = tile0 + t, half_tiles = (F + BM - 1) / BM;
    const int mt = (tile / ntn) * CG + r / BM, up = mt >= half_tiles;
    const int f = (up ? mt - half_tiles : mt) * BM + r % BM, k = (tile % ntn) * BN + c;
    const int U = ntp * blk, lo = t * blk, hi = lo + blk;  // U x groups stays below 2^31 (checked where it is launched)
    int b0 = lo * groups / U, b1 = hi * groups / U;
    while (b0 > 0 && U * b0 / groups > lo) --b0;           // the group whose share holds lo ..
    while (U * (b0 + 1) / groups <= lo) ++b0;
    while (b1 >= groups || U * b1 / groups >= hi) --b1;    // .. to the one whose share holds hi - 1
    after_previous();
    if (f >= F || k >= K) return;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    const float* src = part + ((size_t)t * R + r) * BN + c;
#pragma unroll 8
    for (int b = b0; b <= b1; ++b) {
        const float4 v = __ldcs(reinterpret_cast<const float4*>(src + (size_t)b * R * BN));
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

// rows of 16-bit numbers copied to rows of `ldd` (a multiple of 8), zeros behind the n-th; two matrices in one launch
struct PadJob {
    const uint16_t* src;
    uint16_t* dst;
    long long ld, rows;
};
__global__ void __launch_bounds__(256) k_pad(PadJob a, PadJob b, int ldd, int n) {
    after_previous();
    const int groups = ldd / 8;
    const long long na = a.rows * groups, total = na + b.rows * groups;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const PadJob& j = i < na ? a : b;
        const long long e = i < na ? i : i - na, r = e / groups;
        const int c = (int)(e % groups) * 8;
        uint16_t v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = c + q < n ? j.src[r * j.ld + c + q] : (uint16_t)0;
        uint4 o;
        memcpy(&o, v, 16);
        *reinterpret_cast<uint4*>(j.dst + r * ldd + c) = o;
    }
}

// The forward pass of a few rows (a world or some asking for their next action): the weights' bytes are the work, and
// 128-row tiles would leave it to F / 32 CTAs at most.  One warp an output: it reads row f of Wg and of Wu once, 16 bytes
// a lane (VEC; single numbers where rows start anywhere), the rows of X come from L1.  R rows at a time.  Measured in a
// graph, this and 128-row tiles: 1 x 1024 x 1024 2.1 to 2.5 us and 8.1, 4 rows 5.7 and 8.1 (8 rows took 9.9)
template <class T, int R, bool VEC>
__global__ void __launch_bounds__(256) k_ff_rows(int M, int K, int F, int act, const T* X, long long ldx, const T* W, long long ldw,
                                                 const float* bias, T* __restrict__ h) {
    const int f = (blockIdx.x * 256 + threadIdx.x) >> 5, lane = threadIdx.x & 31;
    after_previous();
    if (f >= F) return;
    const T *wg = W + (size_t)f * ldw, *wu = W + (size_t)(F + f) * ldw;
    for (int m0 = 0; m0 < M; m0 += R) {
        float g[R], u[R];
        if constexpr (VEC) {
            f2 gg[R], uu[R];  // even and odd columns
#pragma unroll
            for (int r = 0; r < R; ++r) gg[r] = uu[r] = 0;
#pragma unroll 4
            for (int k = lane * 8; k < K; k += 256) {
                const uint4 a = *reinterpret_cast<const uint4*>(wg + k), c = *reinterpret_cast<const uint4*>(wu + k);
                const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, cw[4] = {c.x, c.y, c.z, c.w};
                f2 p[4], q[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    p[j] = mk(Half2<T>::unpack(aw[j]));
                    q[j] = mk(Half2<T>::unpack(cw[j]));
                }
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (m0 + r >= M) break;
                    const uint4 x = *reinterpret_cast<const uint4*>(X + (m0 + r) * ldx + k);
                    const uint32_t xw[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const f2 y = mk(Half2<T>::unpack(xw[j]));
                        gg[r] = fma(p[j], y, gg[r]);
                        uu[r] = fma(q[j], y, uu[r]);
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float2 x = un(gg[r]), y = un(uu[r]);
                g[r] = x.x + x.y;
                u[r] = y.x + y.y;
            }
        } else {
#pragma unroll
            for (int r = 0; r < R; ++r) g[r] = u[r] = 0.f;
#pragma unroll 4
            for (int k = lane; k < K; k += 32) {
                const float p = Half2<T>::f(wg[k]), q = Half2<T>::f(wu[k]);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (m0 + r >= M) break;
                    const float y = Half2<T>::f(X[(m0 + r) * ldx + k]);
                    g[r] = fmaf(p, y, g[r]);
                    u[r] = fmaf(q, y, u[r]);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                g[r] += __shfl_xor_sync(0xffffffffu, g[r], o);
                u[r] += __shfl_xor_sync(0xffffffffu, u[r], o);
            }
        }
        const float bg = bias ? bias[f] : 0.f, bu = bias ? bias[F + f] : 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (lane != r || m0 + r >= M) continue;
            f2 a, d;
            const f2 x = all(g[r] + bg);
            if (act == 0) act2<0, false>(x, a, d);
            else if (act == 1) act2<1, false>(x, a, d);
            else if (act == 2) act2<2, false>(x, a, d);
            else act2<3, false>(x, a, d);
            h[(size_t)(m0 + r) * F + f] = Half2<T>::one(un(a).x * (u[r] + bu));
        }
    }
}

// a wait that runs out: on a barrier that nothing arrives at, with no copy or MMA in flight
__global__ void __launch_bounds__(32) k_wait_probe(uint32_t limit) {
    __shared__ uint64_t bar;
    if (threadIdx.x == 0) {
        asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(s32(&bar)));
        if (!wait(&bar, 0u, limit)) atomicExch(&g_err, 1);
    }
}

__global__ void k_take_err() { g_taken = atomicExch(&g_err, 0); }

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

// launches that may start while their predecessor in the stream ends (after_previous); cg CTAs a cluster
template <class... P, class... A>
static cudaError_t go(int cg, void (*k)(P...), dim3 grid, int block, int smem, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = block; cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cg; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = cg > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, k, args...);
}

// the shared-memory limit is a property of (function, device)
template <class T, int MODE, int BN, int CG>
static cudaError_t launch(const Args& P, int groups, cudaStream_t st) {
    static std::once_flag once[64];
    static cudaError_t rc[64];
    constexpr int smem = smem_bytes<MODE, BN, CG>();
    static_assert(smem <= 227 * 1024, "shared memory of a CTA");
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    std::call_once(once[dev], [dev]() {
        rc[dev] = cudaFuncSetAttribute(k_ff<T, MODE, BN, CG>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    });
    if (rc[dev] != cudaSuccess) return rc[dev];
    return go(CG, k_ff<T, MODE, BN, CG>, dim3(groups * CG), Cfg<MODE, BN, CG>::NTH, smem, st, P);
}

// TMA wants rows on 16-byte boundaries
static bool needs_pad(const void* p, long long ld) { return ld % 8 || ((uintptr_t)p & 15); }
static long long up16(long long b) { return (b + 255) & ~255ll; }
static int pad8(int n) { return (n + 7) & ~7; }

constexpr int ROWS_MAX = 4;  // rows up to which the forward pass goes by k_ff_rows

// Columns of B a tile, for `cols` output columns that B has `per` of for each: 256 on pairs of CTAs (cg 2) where that
// gives two of three pairs a tile, else 128 or 64 on single ones, the narrower the fewer tiles there are.  Measured, forward:
// 2048 x 1024 x 1024 (64 pair tiles) 12.0 us on pairs, 15.9 on single CTAs; 1024 x 1024 x 1024 (32) 11.0 and 9.8.  Matrices of
// up to 128 columns on pairs too: backward 65536 x 104 x 1024 233 us, on single CTAs 255.  (Halving the columns of wider
// ones to fill the last wave does not pay, as a half tile takes as long: forward 20000 x 512 x 512 31.7 us, 21.7 without.)
struct Shape {
    int bn, cg;
};
static Shape tile_shape(int M, int cols, int per, int nsm) {
    auto tiles = [&](int rows, int bn) { return (long long)((M + rows - 1) / rows) * ((cols * per + bn - 1) / bn); };
    if (cols * per > 128 && tiles(2 * BM, 256) * 3 >= nsm) return {256, 2};
    if (cols * per > 64 && cols * per <= 128 && tiles(2 * BM, 128) * 3 >= nsm) return {128, 2};
    if (cols * per > 64 && tiles(BM, 128) * 2 > nsm) return {128, 1};
    return {64, 1};
}

struct Plan {
    long long xp, wp, z, db, part, total;  // offsets in the workspace
    bool padx, padw;
    Shape dw;
    int tiles, passes, ntp, groups, blk;
    bool direct;
    Shape dx;
    int dx_tiles, dx_groups;  // dx_groups: 0 where the sum of DX is not cut
};
// Whether a sum of nk chunks for each of `tiles` tiles is cut over `all` groups of CTAs: it saves the idle groups' share of the
// time (a chunk takes some 0.25 us) and costs the partial tiles' way through memory and a launch, some 10 us.
// Measured, backward in a graph: 512 x 104 x 2048 with cut sums 33 us, with whole ones 86 to 114 (dX: 4 tiles, 64 chunks);
// 4096 x 2048 x 2048 with whole ones 182, with cut ones 253 (dW: 2 passes of 64 tiles).
static bool worth_cutting(int nk, long long tiles, int all) { return tiles < all && nk * (all - tiles) >= 40ll * all; }

// DW: passes of at most one tile a group of CTAs (then its share meets two tiles at most)
static Plan plan(int M, int K, int F, const void* X, long long ldx, const void* W, long long ldw, int backward, int nsm) {
    Plan L = {};
    long long o = 0;
    if (!backward && M <= ROWS_MAX) return L;
    L.padx = needs_pad(X, ldx);
    L.padw = needs_pad(W, ldw);
    auto take = [&](long long bytes) { const long long at = o; o += up16(bytes); return at; };
    L.xp = take(L.padx ? (long long)M * pad8(K) * 2 : 0);
    L.wp = take(L.padw ? 2ll * F * pad8(K) * 2 : 0);
    if (backward) {
        L.z = take((long long)M * 2 * pad8(F) * 2);
        L.db = take((long long)nsm * 4 * 2 * F * 4);
        const int nk = (M + BK - 1) / BK;
        // a short sum: small tiles on all SMs, as it is the writing of dW that takes the time
        L.dw = K <= 64 ? Shape{64, 1} : K <= 128 || nk <= 8 ? (nk > DW_BLOCK ? Shape{128, 2} : Shape{128, 1}) : Shape{256, 2};
        const int all = nsm / L.dw.cg;
        L.tiles = 2 * ((F + BM - 1) / BM) / L.dw.cg * ((K + L.dw.bn - 1) / L.dw.bn);
        L.passes = (L.tiles + all - 1) / all;
        L.ntp = (L.tiles + L.passes - 1) / L.passes;
        L.blk = nk < DW_BLOCK ? nk : DW_BLOCK;
        // (rows of dW that start anywhere are written number by number, a row a lane, where no sum follows: not for long)
        L.direct = !worth_cutting(nk, L.ntp, all) && (K % 8 == 0 || nk <= 4);
        // four chunks a share at least
        const long long units = (long long)L.ntp * L.blk;
        L.groups = L.direct ? L.ntp : (int)std::min<long long>(all, std::max<long long>(L.ntp, units / 4));
        long long part = L.direct ? 0 : (long long)(L.groups + L.ntp) * L.dw.cg * BM * L.dw.bn * 4;
        L.dx = tile_shape(M, K, 1, nsm);
        const int nkx = 2 * ((F + BK - 1) / BK);
        if (L.dx.cg == 1) {
            const Shape cut = K <= 64 ? Shape{64, 1} : Shape{128, 1};
            const long long tiles = (long long)((M + BM - 1) / BM) * ((K + cut.bn - 1) / cut.bn);
            if (worth_cutting(nkx, tiles, nsm)) {
                L.dx = cut;
                L.dx_tiles = (int)tiles;
                L.dx_groups = (int)std::min<long long>(nsm, tiles * nkx / 4);
                part = std::max(part, (long long)(L.dx_groups + L.dx_tiles) * BM * cut.bn * 4);
            }
        }
        L.part = take(part);
    }
    L.total = o;
    return L;
}

struct Call {
    int M, K, F, type, act;
    const void* X;
    long long ldx;
    const void* W;
    long long ldw;
    const float* b;
    uint8_t* ws;
    cudaStream_t st;
    int nsm;
    int* err;  // forward: the flag of a wait that runs out, or null for the device's
};

static cudaError_t operands(Call& c, const Plan& L) {
    if (!L.padx && !L.padw) return cudaSuccess;
    const int ldd = pad8(c.K);
    PadJob a = {}, b = {};
    if (L.padx) {
        a = {(const uint16_t*)c.X, (uint16_t*)(c.ws + L.xp), c.ldx, c.M};
        c.X = a.dst;
        c.ldx = ldd;
    }
    if (L.padw) {
        b = {(const uint16_t*)c.W, (uint16_t*)(c.ws + L.wp), c.ldw, 2ll * c.F};
        c.W = b.dst;
        c.ldw = ldd;
    }
    const long long n = (a.rows + b.rows) * (ldd / 8);
    return go(1, k_pad, dim3((unsigned)std::min<long long>((n + 255) / 256, c.nsm * 16)), 256, 0, c.st, a, b, ldd, c.K);
}

template <class T, int MODE>
static cudaError_t pair_tiles(const Call& c, Args P, int* ctas) {
    const Shape sh = tile_shape(c.M, c.F, 2, c.nsm);
    const int tn = sh.bn / 2, rows = BM * sh.cg;
    if (!map2d(&P.a0, c.type, c.X, c.K, c.M, c.ldx, BM) || !map2d(&P.b0, c.type, c.W, c.K, c.F, c.ldw, tn) ||
        !map2d(&P.b1, c.type, (const T*)c.W + c.F * c.ldw, c.K, c.F, c.ldw, tn))
        return cudaErrorInvalidValue;
    P.M = c.M; P.N = c.F; P.F = c.F; P.act = c.act; P.bias = c.b; P.err = c.err;
    P.nk = (c.K + BK - 1) / BK;
    P.up.x = P.up.y = 1.f + TRUNC * (float)((c.K + 15) / 16);
    const int groups = (int)std::min<long long>((long long)((c.M + rows - 1) / rows) * ((c.F + tn - 1) / tn), c.nsm / sh.cg);
    *ctas = groups * sh.cg;
    if (sh.bn == 64) return launch<T, MODE, 64, 1>(P, groups, c.st);
    if (sh.bn == 128) return sh.cg == 2 ? launch<T, MODE, 128, 2>(P, groups, c.st) : launch<T, MODE, 128, 1>(P, groups, c.st);
    return launch<T, MODE, 256, 2>(P, groups, c.st);
}

template <class T>
static cudaError_t forward(Call c, const Plan& L, void* h) {
    if (c.M <= ROWS_MAX) {
        const bool vec = c.K % 8 == 0 && !needs_pad(c.X, c.ldx) && !needs_pad(c.W, c.ldw);
        auto rows = [&](auto k) {
            return go(1, k, dim3((c.F + 7) / 8), 256, 0, c.st, c.M, c.K, c.F, c.act, (const T*)c.X, c.ldx, (const T*)c.W, c.ldw, c.b,
                      (T*)h);
        };
        if (c.M == 1) return vec ? rows(k_ff_rows<T, 1, true>) : rows(k_ff_rows<T, 1, false>);
        return vec ? rows(k_ff_rows<T, 4, true>) : rows(k_ff_rows<T, 4, false>);
    }
    cudaError_t e = operands(c, L);
    if (e != cudaSuccess) return e;
    Args P = {};
    P.out = h; P.ldo = c.F;
    P.vec = c.F % 8 == 0 && ((uintptr_t)h & 15) == 0;
    int ctas;
    return pair_tiles<T, FWD>(c, P, &ctas);
}

// sums partial tiles (of dX as of dW); the last blocks sum db where it is given
template <class T, class O, int BN, int CG>
static cudaError_t sum_tiles(const Call& c, const float* part, O* out, int rows, int tile0, int ntp, int blk, int groups,
                             const float* db_part, float* db, int db_rows) {
    if ((long long)ntp * blk * (groups + 1) >= (1ll << 31)) return cudaErrorInvalidValue;
    const int x = CG * BM * BN / 4 / 256;
    const dim3 grid(x, ntp + (db ? ((2 * c.F + 7) / 8 + x - 1) / x : 0));
    if (grid.y > 65535) return cudaErrorInvalidValue;
    return go(1, k_dw_sum<O, BN, CG>, grid, 256, 0, c.st, part, out, rows, c.K, tile0, ntp, blk, groups, (c.K + BN - 1) / BN, db_part,
              db, db_rows);
}

template <class T, int BN, int CG>
static cudaError_t dw_passes(const Call& c, const Plan& L, Args P, void* dw, int dw_type, const float* db_part, float* db, int db_rows) {
    P.blk = L.blk;
    P.direct = L.direct;
    P.out32 = dw_type == 0;
    P.out = L.direct ? dw : c.ws + L.part;
    P.vec = c.K % 8 == 0 && ((uintptr_t)dw & 15) == 0;
    const float* part = (const float*)P.out;
    for (int t0 = 0; t0 < L.tiles; t0 += L.ntp) {
        P.tile0 = t0;
        P.ntp = std::min(L.ntp, L.tiles - t0);
        const int groups = L.direct ? P.ntp : (int)std::min<long long>((long long)P.ntp * L.blk, L.groups);
        cudaError_t e = launch<T, DW, BN, CG>(P, groups, c.st);
        if (e != cudaSuccess) return e;
        if (L.direct) continue;
        e = dw_type == 0 ? sum_tiles<T, float, BN, CG>(c, part, (float*)dw, c.F, t0, P.ntp, L.blk, groups, db_part, db, db_rows)
                         : sum_tiles<T, T, BN, CG>(c, part, (T*)dw, c.F, t0, P.ntp, L.blk, groups, db_part, db, db_rows);
        if (e != cudaSuccess) return e;
        db = nullptr;  // with the first pass
    }
    return db ? sum_tiles<T, T, 64, 1>(c, nullptr, (T*)nullptr, c.F, 0, 0, 1, 1, db_part, db, db_rows) : cudaSuccess;
}

template <class T>
static cudaError_t backward(Call c, const Plan& L, const void* dh, void* dx, void* dw, int dw_type, float* db) {
    cudaError_t e = operands(c, L);
    if (e != cudaSuccess) return e;
    const int Fp = pad8(c.F);
    T* z = (T*)(c.ws + L.z);
    const T* Wu = (const T*)c.W + c.F * c.ldw;
    int ctas;
    {   // z = [dg | du] and the column sums
        Args P = {};
        P.out = z; P.ldo = 2 * Fp;
        P.dh = dh;
        P.vec = c.F % 8 == 0 && ((uintptr_t)dh & 15) == 0;
        P.db = db ? (float*)(c.ws + L.db) : nullptr;
        e = P.vec ? pair_tiles<T, DZ>(c, P, &ctas) : pair_tiles<T, DZU>(c, P, &ctas);
        if (e != cudaSuccess) return e;
    }
    const float* db_part = (const float*)(c.ws + L.db);
    if (dx) {
        Args P = {};
        if (!map2d(&P.a0, c.type, z, c.F, c.M, 2 * Fp, BM) || !map2d(&P.a1, c.type, z + Fp, c.F, c.M, 2 * Fp, BM) ||
            !map2d(&P.b0, c.type, c.W, c.K, c.F, c.ldw, BK) || !map2d(&P.b1, c.type, Wu, c.K, c.F, c.ldw, BK))
            return cudaErrorInvalidValue;
        P.M = c.M; P.N = c.K; P.F = c.F;
        P.nk = 2 * ((c.F + BK - 1) / BK);
        P.out = dx; P.ldo = c.K;
        P.vec = c.K % 8 == 0 && ((uintptr_t)dx & 15) == 0;
        const Shape sh = L.dx;
        if (L.dx_groups) {
            P.blk = P.nk;
            P.ntp = L.dx_tiles;
            P.out = c.ws + L.part;
            e = sh.bn == 64 ? launch<T, DXS, 64, 1>(P, L.dx_groups, c.st) : launch<T, DXS, 128, 1>(P, L.dx_groups, c.st);
            if (e != cudaSuccess) return e;
            const float* part = (const float*)P.out;
            // as dW's gate half: M rows
            e = sh.bn == 64 ? sum_tiles<T, T, 64, 1>(c, part, (T*)dx, c.M, 0, P.ntp, P.blk, L.dx_groups, nullptr, nullptr, 0)
                            : sum_tiles<T, T, 128, 1>(c, part, (T*)dx, c.M, 0, P.ntp, P.blk, L.dx_groups, nullptr, nullptr, 0);
        } else {
            const int rows = BM * sh.cg;
            const int groups = (int)std::min<long long>((long long)((c.M + rows - 1) / rows) * ((c.K + sh.bn - 1) / sh.bn), c.nsm / sh.cg);
            e = sh.bn == 64    ? launch<T, DX, 64, 1>(P, groups, c.st)
                : sh.bn == 128 ? (sh.cg == 2 ? launch<T, DX, 128, 2>(P, groups, c.st) : launch<T, DX, 128, 1>(P, groups, c.st))
                               : launch<T, DX, 256, 2>(P, groups, c.st);
        }
        if (e != cudaSuccess) return e;
    }
    if (dw) {
        Args P = {};
        if (!map2d(&P.a0, c.type, z, c.F, c.M, 2 * Fp, BK) || !map2d(&P.a1, c.type, z + Fp, c.F, c.M, 2 * Fp, BK) ||
            !map2d(&P.b0, c.type, c.X, c.K, c.M, c.ldx, BK))
            return cudaErrorInvalidValue;
        P.M = c.M; P.N = c.K; P.F = c.F;
        P.nk = (c.M + BK - 1) / BK;
        return L.dw.bn == 64    ? dw_passes<T, 64, 1>(c, L, P, dw, dw_type, db_part, db, ctas * 4)
               : L.dw.bn == 256 ? dw_passes<T, 256, 2>(c, L, P, dw, dw_type, db_part, db, ctas * 4)
               : L.dw.cg == 2   ? dw_passes<T, 128, 2>(c, L, P, dw, dw_type, db_part, db, ctas * 4)
                                : dw_passes<T, 128, 1>(c, L, P, dw, dw_type, db_part, db, ctas * 4);
    }
    if (db) e = sum_tiles<T, T, 64, 1>(c, nullptr, (T*)nullptr, c.F, 0, 0, 1, 1, db_part, db, ctas * 4);
    return e;
}

// a gated layer of the wide policies' rollout: bf16, rows and weights on 16-byte boundaries (K a multiple of 8); err: the
// env's flag
static cudaError_t policy_layer(int M, int K, int F, int act, const __nv_bfloat16* X, const __nv_bfloat16* W, const float* b,
                                __nv_bfloat16* h, int nsm, int* err, cudaStream_t st) {
    if (needs_pad(X, K) || needs_pad(W, K)) return cudaErrorInvalidValue;
    const Call c = {M, K, F, 1, act, X, K, W, K, b, nullptr, st, nsm, err};
    return forward<__nv_bfloat16>(c, plan(M, K, F, X, K, W, K, 0, nsm), h);
}

// tile indices are 32-bit
static bool shape_ok(int M, int K, int F) {
    return M >= 0 && K >= 1 && F >= 1 && M <= (1 << 30) && K <= (1 << 20) && F <= (1 << 20) &&
           ((long long)M / BM + 1) * ((long long)std::max(K, F) / 128 + 1) < (1ll << 30);
}

// shared argument checks; 0 when the call can run
static int check(const char* who, int M, int K, int F, int type, int act, const void* X, long long ldx, const void* W,
                 long long ldw, const float* b, const void* ws, long long ws_size, int backward, Plan* L, int* nsm) {
    auto bad = [&](const char* what) { set_error(-22, who, what); return -22; };
    if (!shape_ok(M, K, F)) return bad("invalid shape");
    if (type != 1 && type != 2) return bad("type must be 1 (bf16) or 2 (fp16)");
    if (act < 0 || act > 3) return bad("activation must be 0 tanh, 1 ELU, 2 SiLU or 3 GELU");
    if ((ldx < K && M > 1) || ldw < K || ldx > (1ll << 36) || ldw > (1ll << 36)) return bad("row stride below K or too long");
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
    *L = plan(M, K, F, X, ldx, W, ldw, backward, *nsm);
    if (L->total > 0 && (!ws || ((uintptr_t)ws & 255) || ws_size < L->total))
        return bad("workspace too small or not 256-byte aligned");
    return 0;
}

}  // namespace g1ff

extern "C" {

long long g1_gated_ff_workspace(int M, int K, int F, const void* X, long long ldx, const void* W, long long ldw,
                                int backward) {
    if (!g1ff::shape_ok(M, K, F)) return 0;
    int dev = 0, nsm = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&nsm, cudaDevAttrMultiProcessorCount, dev);
    return g1ff::plan(M, K, F, X, M == 1 ? g1ff::pad8(K) : ldx, W, ldw, backward, nsm).total;
}

int g1_gated_ff(int M, int K, int F, int type, int act, const void* X, long long ldx, const void* W, long long ldw,
                const float* b, void* h, void* ws, long long ws_size, void* stream) {
    g1ff::Plan L;
    g1ff::Call c = {M, K, F, type, act, X, M == 1 ? g1ff::pad8(K) : ldx, W, ldw, b, (uint8_t*)ws, (cudaStream_t)stream, 148,
                    nullptr};
    const int rc = g1ff::check("g1_gated_ff", M, K, F, type, act, X, c.ldx, W, ldw, b, ws, ws_size, 0, &L, &c.nsm);
    if (rc) return rc;
    if (M > 0 && (!h || ((uintptr_t)h & 1))) { set_error(-22, "g1_gated_ff", "null or misaligned h"); return -22; }
    if (M == 0) return 0;
    const cudaError_t e = type == 1 ? g1ff::forward<__nv_bfloat16>(c, L, h) : g1ff::forward<__half>(c, L, h);
    if (e != cudaSuccess) { set_error((int)e, "g1_gated_ff", cudaGetErrorString(e)); return -1; }
    return 0;
}

int g1_gated_ff_backward(int M, int K, int F, int type, int act, const void* dh, const void* X, long long ldx, const void* W,
                         long long ldw, const float* b, void* dx, void* dw, int dw_type, float* db, void* ws, long long ws_size,
                         void* stream) {
    g1ff::Plan L;
    g1ff::Call c = {M, K, F, type, act, X, M == 1 ? g1ff::pad8(K) : ldx, W, ldw, b, (uint8_t*)ws, (cudaStream_t)stream, 148,
                    nullptr};
    const int rc = g1ff::check("g1_gated_ff_backward", M, K, F, type, act, X, c.ldx, W, ldw, b, ws, ws_size, 1, &L, &c.nsm);
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

// Test entry (not part of the public header): a wait with a limit of `limit` tries that runs out and says so
// (g1_gated_ff_status).  Returns the CUDA status.
int g1_gated_ff_test_wait(unsigned limit, void* stream) {
    g1ff::k_wait_probe<<<1, 32, 0, (cudaStream_t)stream>>>(limit);
    return (int)cudaGetLastError();
}

int g1_gated_ff_status(void) {
    static std::mutex mu;  // g_taken is one a device
    std::lock_guard<std::mutex> lk(mu);
    // the calls of every stream are over: those that other threads make from here on are the next status call's
    if (cudaDeviceSynchronize() != cudaSuccess) return -1;
    g1ff::k_take_err<<<1, 1>>>();
    int v = 0;
    if (cudaGetLastError() != cudaSuccess || cudaMemcpyFromSymbol(&v, g1ff::g_taken, sizeof v) != cudaSuccess) return -1;
    return v;
}

}  // extern "C"
