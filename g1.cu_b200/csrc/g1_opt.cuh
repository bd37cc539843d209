// g1_opt.cuh -- the end of the trainer's update on the GPU: the global gradient norm over all of a
// network's tensors, clipping, and the Adam step that takes the clip factor along (the reference trainer's
// clip_grad_norm_ and optimiser step, scripts/ppo_fused.py:77-78,121-140).
//
//   norm = sqrt(sum over tensors and elements of g^2),   c = min(1, max_norm / (norm + 1e-6))
//   clip:  g <- c g                        (in place)
//   Adam:  g' = c g,  m <- m + (1 - b1)(g' - m),  v <- b2 v + (1 - b2) g'^2,
//          p <- (1 - lr wd) p - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Both are bound by memory: clipping N fp32 numbers reads and writes 8N bytes, the Adam step reads g, p, m, v
// and writes p, m, v, 28N bytes; the clip factor needs the whole norm first, so what does not stay in L2 of g is
// read twice.  The squares are summed in fp64: an fp32 square overflows from 1.8e19 and vanishes below 1e-23, and
// a sum of 10^8 of them loses digits; the conversions stay below the time of the loads.
//
// A tensor is cut into chunks, and a chunk's tensor is found by a search in the list, so one launch serves any number of
// tensors.  Up to TAB tensors travel in the kernel's parameters; longer lists are laid into the workspace by k_table,
// whose parameters carry TAB_BIG entries a launch.  Parameters are copied at launch or capture, so a captured call
// holds no host memory.
//
// k_norm's block sums go to the workspace and are added up in one order (by every block of k_apply, or once by k_total where
// k_apply has more blocks than fit): no atomics, the same bits for the same list of lengths and alignments on the same kind
// of card, no counter that a call would have to clear.  k_apply takes the last chunk first: what k_norm read last is
// still in L2.
//
// Networks of up to CL * R chunks of CH_SMALL run as one launch of one 16-CTA cluster (k_small): every thread reads its
// numbers once and holds them in registers, the block sums cross in distributed shared memory behind the hardware's
// cluster barrier, and the results are written.
//
// Measured on one B200, replayed from a graph (floor: the bytes at the measured 6552 GB/s; memory of the smaller ones stays
// in L2 between replays):
//   clip   99387 fp32 in 9 tensors      7 us (12.4 when each chunk was loaded for the norm and again for the clip)
//          3e6 bf16 in 300 tensors     14 us; floor 1.8
//          2.7e8 fp32 in 40 tensors   496 us; floor 328, 491 with the second read that 1 GB needs
//   Adam   99387                       12 us
//          2270267 in 17 tensors       14 us; floor 9.7
//          6.7e7, bf16 gradients      318 to 353 us, by process and box; floor 266, 287 with the second read
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <algorithm>
#include <new>
#include <vector>

namespace g1opt {

constexpr int THREADS = 256;          // threads a block of the two-launch path
// resident blocks an SM that k_norm and k_apply are compiled for: what bounds them is the loads in flight (with the
// registers that the compiler took, 48 a thread, clipping 2.7e8 numbers took 605 us, with these 496)
constexpr int NORM_CTAS = 4, ADAM_CTAS = 3, CLIP_CTAS = 6;
constexpr int UNROLL = 4;
constexpr int CL = 16, CL_THREADS = 512, R = 4;  // the small path: CTAs of its cluster, chunks a CTA holds
constexpr int CH_SMALL = 2048, CH_BIG = 8192;    // numbers a chunk
static_assert(CH_SMALL == 4 * CL_THREADS, "four numbers a thread");
constexpr int MAX_PARTS = 2048;
constexpr int TAB = 48, TAB_BIG = 448;

struct Entry {
    void* g;
    float *p, *m, *v;
    long long n, chunk0;  // numbers; index of the tensor's first chunk
    int type, index;      // 0 fp32, 1 bf16, 2 fp16; place in the caller's list
    int head, pad;        // numbers before the first 128-byte boundary (of g, of p for Adam): part of the first chunk
};
template <int N>
struct Table {
    Entry e[N];
};
struct Args {
    const Entry* table;   // in the workspace, or null: the table is in the parameters
    int n, ch, nparts, adam;
    long long chunks;
    double max_norm, b1d, b2d;
    float omb1, b2, omb2, eps, lr, wd;
    const float* lr_dev;
    long long* steps;
    float* norm;
    double* part;
    float2* bias;         // per tensor: 1 / (1 - b1^t), 1 / sqrt(1 - b2^t)
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ void from_f(float x, float& o) { o = x; }
__device__ __forceinline__ void from_f(float x, __nv_bfloat16& o) { o = __float2bfloat16_rn(x); }
__device__ __forceinline__ void from_f(float x, __half& o) { o = __float2half_rn(x); }

template <class T, int N>
struct alignas(sizeof(T) * N) Vec {
    T x[N];
};

// the last entry whose first chunk is <= c (empty tensors are not in the list).  A table in the kernel's parameters is
// searched by every thread for itself; one in memory by the block, whose threads look at all entries at once
__device__ __forceinline__ int find(const Entry* t, int n, long long c, bool in_memory) {
    if (in_memory) {
        int at = -1;
        for (int i = 0; i < n; i += blockDim.x)
            at += __syncthreads_count(i + threadIdx.x < n && t[min(i + (int)threadIdx.x, n - 1)].chunk0 <= c);
        return at;
    }
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t[mid].chunk0 <= c) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// numbers [lo, lo + cnt) of a tensor's chunk: from the second on chunks start on 128-byte boundaries, so that only a
// tensor's ends take accesses of single numbers (with chunks cut anywhere each one waited for its first few numbers
// before the rest: clipping 2.7e8 of them took 763 instead of 627 us)
__device__ __forceinline__ long long chunk_of(const Entry& e, long long c, int ch, int& cnt) {
    const long long j = c - e.chunk0, lo = j ? e.head + j * ch : 0, hi = min(e.n, e.head + (j + 1) * ch);
    cnt = (int)(hi - lo);
    return lo;
}

// A launch may start while the one before it in the stream ends: wait here before the first access to memory.  Loads
// are ordinary ones: data of read-only ones would have to stay as it is for as long as the kernel is resident
__device__ __forceinline__ void after_previous() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
}

// numbers before the first 128-byte boundary: from there a warp's accesses are whole lines
template <class T>
__device__ __forceinline__ int head_of(const T* p, int cnt) {
    const int h = (int)(-(uintptr_t)p & 127) / (int)sizeof(T);
    return h < cnt ? h : cnt;
}

template <class T>
__device__ __forceinline__ double sumsq(const T* p, int cnt) {
    constexpr int N = 16 / sizeof(T);
    const int tid = threadIdx.x, nt = blockDim.x;
    const int head = head_of(p, cnt), nv = (cnt - head) / N, tail = head + nv * N;
    double acc = 0.0;
    if (tid < head) { const double x = to_f(p[tid]); acc += x * x; }
    if (tid < cnt - tail) { const double x = to_f(p[tail + tid]); acc += x * x; }
    const Vec<T, N>* q = reinterpret_cast<const Vec<T, N>*>(p + head);
#pragma unroll UNROLL
    for (int i = tid; i < nv; i += nt) {
        const Vec<T, N> w = q[i];
#pragma unroll
        for (int k = 0; k < N; ++k) { const double x = to_f(w.x[k]); acc = fma(x, x, acc); }
    }
    return acc;
}

template <class T>
__device__ __forceinline__ void scale(T* p, int cnt, float c) {
    constexpr int N = 16 / sizeof(T);
    const int tid = threadIdx.x, nt = blockDim.x;
    const int head = head_of(p, cnt), nv = (cnt - head) / N, tail = head + nv * N;
    if (tid < head) from_f(to_f(p[tid]) * c, p[tid]);
    if (tid < cnt - tail) from_f(to_f(p[tail + tid]) * c, p[tail + tid]);
    Vec<T, N>* q = reinterpret_cast<Vec<T, N>*>(p + head);
#pragma unroll UNROLL
    for (int i = tid; i < nv; i += nt) {
        Vec<T, N> w = q[i];
#pragma unroll
        for (int k = 0; k < N; ++k) from_f(to_f(w.x[k]) * c, w.x[k]);
        q[i] = w;
    }
}

struct Coef {
    float c, omb1, b2, omb2, eps, decay, a, rb2;  // decay = 1 - lr wd, a = lr / (1 - b1^t), rb2 = 1/sqrt(1 - b2^t)
};
__device__ __forceinline__ void adam1(float g, float& p, float& m, float& v, const Coef& k) {
    g *= k.c;
    m = fmaf(k.omb1, g - m, m);
    v = fmaf(k.b2, v, k.omb2 * g * g);
    p = fmaf(p, k.decay, -k.a * (m / fmaf(sqrtf(v), k.rb2, k.eps)));
}

template <class T>
__device__ __forceinline__ void adam(const T* g, float* __restrict__ p, float* __restrict__ m, float* __restrict__ v, int cnt,
                                     const Coef& k) {
    const int tid = threadIdx.x, nt = blockDim.x;
    int head = head_of(p, cnt);
    // 4-wide where all four pointers reach their boundary after the same number of elements
    const bool vec = ((((uintptr_t)(p + head)) | ((uintptr_t)(m + head)) | ((uintptr_t)(v + head))) & 15) == 0 &&
                     ((uintptr_t)(g + head) & (4 * sizeof(T) - 1)) == 0;
    if (!vec) head = cnt;
    const int nv = (cnt - head) / 4, tail = head + nv * 4;
    for (int i = tid; i < head; i += nt) adam1(to_f(g[i]), p[i], m[i], v[i], k);
    for (int i = tail + tid; i < cnt; i += nt) adam1(to_f(g[i]), p[i], m[i], v[i], k);
    const Vec<T, 4>* gq = reinterpret_cast<const Vec<T, 4>*>(g + head);
    float4* pq = reinterpret_cast<float4*>(p + head);
    float4* mq = reinterpret_cast<float4*>(m + head);
    float4* vq = reinterpret_cast<float4*>(v + head);
#pragma unroll 2
    for (int i = tid; i < nv; i += nt) {
        const Vec<T, 4> gw = gq[i];
        float4 pw = __ldcs(pq + i), mw = __ldcs(mq + i), vw = __ldcs(vq + i);
        adam1(to_f(gw.x[0]), pw.x, mw.x, vw.x, k);
        adam1(to_f(gw.x[1]), pw.y, mw.y, vw.y, k);
        adam1(to_f(gw.x[2]), pw.z, mw.z, vw.z, k);
        adam1(to_f(gw.x[3]), pw.w, mw.w, vw.w, k);
        __stcs(pq + i, pw);
        __stcs(mq + i, mw);
        __stcs(vq + i, vw);
    }
}

// the sum over a block, the same for every thread; sh: 33 doubles
__device__ __forceinline__ double block_sum(double x, double* sh) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if (lane == 0) sh[w] = x;
    __syncthreads();
    if (w == 0) {
        double y = lane < nw ? sh[lane] : 0.0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
        if (lane == 0) sh[32] = y;
    }
    __syncthreads();
    return sh[32];
}

// advances the step counters and leaves the bias corrections of the step being taken
__device__ __forceinline__ void advance(const Args& A, const Entry* tab, int first, int stride) {
    for (int t = first; t < A.n; t += stride) {
        long long* p = A.steps + tab[t].index;
        const long long s = *p + 1;
        *p = s;
        A.bias[t] = make_float2((float)(1.0 / (1.0 - pow(A.b1d, (double)s))), (float)(1.0 / sqrt(1.0 - pow(A.b2d, (double)s))));
    }
}

// the blocks take the chunks in turn, so that all of them read one stretch of memory at a time (runs of neighbours a block
// need one search only, but measured 756 us where this takes 698: 2.7e8 fp32 numbers, norm and clip)
__device__ __forceinline__ double norm_chunks(const Args& A, const Entry* tab) {
    double acc = 0.0;
    for (long long c = blockIdx.x; c < A.chunks; c += gridDim.x) {
        const Entry& e = tab[find(tab, A.n, c, A.table)];
        int cnt;
        const long long off = chunk_of(e, c, A.ch, cnt);
        if (e.type == 0) acc += sumsq((const float*)e.g + off, cnt);
        else if (e.type == 1) acc += sumsq((const __nv_bfloat16*)e.g + off, cnt);
        else acc += sumsq((const __half*)e.g + off, cnt);
    }
    return acc;
}

__device__ __forceinline__ float clip_factor(const Args& A, double total, bool write) {
    const double norm = sqrt(total);
    if (write) *A.norm = (float)norm;
    const double c = isinf(A.max_norm) ? 1.0 : A.max_norm / (norm + 1e-6);  // no limit: not inf / inf
    return c > 1.0 ? 1.f : (float)c;  // a NaN norm stays NaN, as in torch
}

__device__ __forceinline__ Coef coef_of(const Args& A, float c, float lr) {
    Coef k;
    k.c = c; k.omb1 = A.omb1; k.b2 = A.b2; k.omb2 = A.omb2; k.eps = A.eps;
    k.decay = 1.f - lr * A.wd;
    return k;
}

template <bool ADAM>
__device__ __forceinline__ void apply_chunk(const Args& A, const Entry* tab, float c, long long ch) {
    const float lr = ADAM ? (A.lr_dev ? *A.lr_dev : A.lr) : 0.f;
    const int t = find(tab, A.n, ch, A.table);
    const Entry& e = tab[t];
    int cnt;
    const long long off = chunk_of(e, ch, A.ch, cnt);
    if (ADAM) {
        Coef k = coef_of(A, c, lr);
        const float2 b = A.bias[t];
        k.a = lr * b.x;
        k.rb2 = b.y;
        if (e.type == 0) adam((const float*)e.g + off, e.p + off, e.m + off, e.v + off, cnt, k);
        else if (e.type == 1) adam((const __nv_bfloat16*)e.g + off, e.p + off, e.m + off, e.v + off, cnt, k);
        else adam((const __half*)e.g + off, e.p + off, e.m + off, e.v + off, cnt, k);
    } else {
        if (e.type == 0) scale((float*)e.g + off, cnt, c);
        else if (e.type == 1) scale((__nv_bfloat16*)e.g + off, cnt, c);
        else scale((__half*)e.g + off, cnt, c);
    }
}

// 16 entries a block (one reading them all takes 10 us: each lane of a warp wants other words of the parameters, which
// come one at a time)
__global__ void k_table(const __grid_constant__ Table<TAB_BIG> T, int count, Entry* dst) {
    static_assert(sizeof(Entry) % 8 == 0, "words of 8 bytes");
    after_previous();
    constexpr int W = sizeof(Entry) / 8;
    const unsigned long long* src = reinterpret_cast<const unsigned long long*>(T.e);
    const int lo = blockIdx.x * 16 * W, hi = min(lo + 16 * W, count * W);
    for (int i = lo + threadIdx.x; i < hi; i += 32) reinterpret_cast<unsigned long long*>(dst)[i] = src[i];
}

__global__ void __launch_bounds__(THREADS, NORM_CTAS) k_norm(const __grid_constant__ Args A, const __grid_constant__ Table<TAB> T) {
    __shared__ double sh[33];
    const Entry* tab = A.table ? A.table : T.e;
    after_previous();
    const double s = block_sum(norm_chunks(A, tab), sh);
    if (threadIdx.x == 0) A.part[blockIdx.x] = s;
    if (A.adam) advance(A, tab, blockIdx.x * THREADS + threadIdx.x, gridDim.x * THREADS);
}

// the norm and the clip factor (at part[MAX_PARTS]) from the block sums, for lists that k_apply takes in many blocks
__global__ void __launch_bounds__(1024) k_total(const __grid_constant__ Args A) {
    __shared__ double sh[33];
    after_previous();
    double x = 0.0;
    for (int i = threadIdx.x; i < A.nparts; i += 1024) x += A.part[i];
    const double total = block_sum(x, sh);
    if (threadIdx.x == 0) *reinterpret_cast<float*>(A.part + MAX_PARTS) = clip_factor(A, total, true);
}

// One block a chunk, the last chunk first.  SUM: every block adds the block sums up by itself.
template <bool SUM, bool ADAM>
__global__ void __launch_bounds__(THREADS, ADAM ? ADAM_CTAS : CLIP_CTAS) k_apply(const __grid_constant__ Args A, const __grid_constant__ Table<TAB> T) {
    __shared__ double sh[33];
    const Entry* tab = A.table ? A.table : T.e;
    after_previous();
    float c;
    if (SUM) {
        double x = 0.0;
#pragma unroll 4
        for (int i = threadIdx.x; i < A.nparts; i += THREADS) x += A.part[i];
        const double total = block_sum(x, sh);
        c = clip_factor(A, total, blockIdx.x == 0 && threadIdx.x == 0);
    } else {
        c = *reinterpret_cast<const float*>(A.part + MAX_PARTS);
    }
    if (blockIdx.x < A.chunks) apply_chunk<ADAM>(A, tab, c, A.chunks - 1 - blockIdx.x);
}

// four neighbours of a tensor, the first `cnt` of them inside it; a wide access where the address and cnt allow it
template <class T>
__device__ __forceinline__ void load4(const T* p, int cnt, float* x) {
    if (cnt >= 4 && ((uintptr_t)p & (4 * sizeof(T) - 1)) == 0) {
        const Vec<T, 4> v = *reinterpret_cast<const Vec<T, 4>*>(p);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = to_f(v.x[k]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = k < cnt ? to_f(p[k]) : 0.f;
    }
}
template <class T>
__device__ __forceinline__ void store4(T* p, int cnt, const float* x) {
    if (cnt >= 4 && ((uintptr_t)p & (4 * sizeof(T) - 1)) == 0) {
        Vec<T, 4> v;
#pragma unroll
        for (int k = 0; k < 4; ++k) from_f(x[k], v.x[k]);
        *reinterpret_cast<Vec<T, 4>*>(p) = v;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k < cnt) from_f(x[k], p[k]);
    }
}

template <bool ADAM>
__global__ void __launch_bounds__(CL_THREADS) k_small(const __grid_constant__ Args A, const __grid_constant__ Table<TAB> T) {
    __shared__ double sh[33];
    __shared__ double mine;
    __shared__ int s_at[R];
    const Entry* tab = A.table ? A.table : T.e;
    const int r = blockIdx.x, tid = threadIdx.x;  // the grid is one cluster
    after_previous();
    if (A.table) {
        for (int j = 0; j < R; ++j) {
            const int at = find(tab, A.n, r + j * CL, true);
            if (tid == 0) s_at[j] = at;
        }
    } else if (tid < R) {
        s_at[tid] = find(tab, A.n, r + tid * CL, false);
    }
    __syncthreads();
    float g[R][4], p[ADAM ? R : 1][4], m[ADAM ? R : 1][4], v[ADAM ? R : 1][4];
    long long off[R];
    int cnt[R];
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const Entry& e = tab[max(s_at[j], 0)];
        off[j] = (r + j * CL - e.chunk0) * CH_SMALL + 4 * tid;
        cnt[j] = r + j * CL < A.chunks ? (int)min(4ll, max(0ll, e.n - off[j])) : 0;
        if (e.type == 0) load4((const float*)e.g + off[j], cnt[j], g[j]);
        else if (e.type == 1) load4((const __nv_bfloat16*)e.g + off[j], cnt[j], g[j]);
        else load4((const __half*)e.g + off[j], cnt[j], g[j]);
        if (ADAM) {
            load4(e.p + off[j], cnt[j], p[ADAM ? j : 0]);
            load4(e.m + off[j], cnt[j], m[ADAM ? j : 0]);
            load4(e.v + off[j], cnt[j], v[ADAM ? j : 0]);
        }
    }
    if (ADAM) advance(A, tab, r * CL_THREADS + (CL_THREADS - 1 - tid), CL * CL_THREADS);
    double acc = 0.0;
#pragma unroll
    for (int j = 0; j < R; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) { const double x = g[j][k]; acc = fma(x, x, acc); }
    const double s = block_sum(acc, sh);
    if (tid == 0) mine = s;
    __syncthreads();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    double total = 0.0;
#pragma unroll
    for (int k = 0; k < CL; ++k) {
        uint32_t a = (uint32_t)__cvta_generic_to_shared(&mine), remote;
        double x;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(a), "r"(k));
        asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(x) : "r"(remote) : "memory");
        total += x;
    }
    // no CTA leaves before the others have read its sum
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    const float c = clip_factor(A, total, r == 0 && tid == 0);
    const float lr = ADAM ? (A.lr_dev ? *A.lr_dev : A.lr) : 0.f;
    Coef k = coef_of(A, c, lr);
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const Entry& e = tab[max(s_at[j], 0)];
        if (cnt[j] == 0) continue;
        if constexpr (ADAM) {
            const float2 b = A.bias[max(s_at[j], 0)];
            k.a = lr * b.x;
            k.rb2 = b.y;
#pragma unroll
            for (int i = 0; i < 4; ++i) adam1(g[j][i], p[j][i], m[j][i], v[j][i], k);
            store4(e.p + off[j], cnt[j], p[j]);
            store4(e.m + off[j], cnt[j], m[j]);
            store4(e.v + off[j], cnt[j], v[j]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) g[j][i] *= c;
            if (e.type == 0) store4((float*)e.g + off[j], cnt[j], g[j]);
            else if (e.type == 1) store4((__nv_bfloat16*)e.g + off[j], cnt[j], g[j]);
            else store4((__half*)e.g + off[j], cnt[j], g[j]);
        }
    }
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// a launch that may start while its predecessor in the stream ends (after_previous), in clusters of `cl` CTAs
template <class... P, class... A>
static cudaError_t go(int cl, void (*k)(P...), int grid, int block, cudaStream_t st, const A&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = block; cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cl; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = cl > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, k, args...);
}

// whether a 16-CTA cluster of k_small fits on the current device (asked once a device)
template <bool ADAM>
static bool cluster_fits(int dev) {
    static std::once_flag once[64];
    static bool ok[64];
    if (dev < 0 || dev >= 64) return false;
    std::call_once(once[dev], [dev]() {
        ok[dev] = false;
        if (cudaFuncSetAttribute(k_small<ADAM>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = CL; cfg.blockDim = CL_THREADS;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = CL; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
        cfg.attrs = at; cfg.numAttrs = 1;
        int n = 0;
        ok[dev] = cudaOccupancyMaxActiveClusters(&n, k_small<ADAM>, &cfg) == cudaSuccess && n >= 1;
        (void)cudaGetLastError();
    });
    return ok[dev];
}

static size_t ws_bytes(int n) {
    return (MAX_PARTS + 1) * sizeof(double) + (size_t)n * (sizeof(float2) + sizeof(Entry)) + 64;
}

// two ranges of memory of one call may not share a byte: they are written by different blocks
static bool overlap(std::vector<std::pair<uintptr_t, uintptr_t>>& r) {
    std::sort(r.begin(), r.end());
    for (size_t i = 1; i < r.size(); ++i)
        if (r[i].first < r[i - 1].second) return true;
    return false;
}

static int run(const char* who, int n, void* const* g, const int* types, float* const* p, float* const* m,
               float* const* v, const long long* counts, long long* steps, Args A, void* ws, long long ws_size,
               cudaStream_t st) {
    auto bad = [&](const char* what) { set_error(-22, who, what); return -22; };
    if (n < 0) return bad("negative number of tensors");
    if (!A.norm) return bad("no place for the norm");
    if (!(A.max_norm >= 0.0)) return bad("max_norm must be a number >= 0");
    if (n > 0 && (!g || !types || !counts)) return bad("null table");
    if (A.adam && n > 0 && (!p || !m || !v || !steps)) return bad("null table");
    if (!ws || ((uintptr_t)ws & 15) || ws_size < (long long)ws_bytes(n)) return bad("workspace too small or not 16-byte aligned");
    if (((uintptr_t)A.norm & 3) || ((uintptr_t)steps & 7)) return bad("misaligned pointer");
    std::vector<Entry> tab;
    std::vector<std::pair<uintptr_t, uintptr_t>> ranges;
    long long total = 0;
    tab.reserve(n);
    ranges.reserve((size_t)n * (A.adam ? 4 : 1));
    for (int i = 0; i < n; ++i) {
        if (counts[i] < 0 || counts[i] > (1ll << 40)) return bad("bad tensor length");
        if (types[i] < 0 || types[i] > 2) return bad("bad gradient type (0 fp32, 1 bf16, 2 fp16)");
        if (counts[i] == 0) continue;
        const int es = types[i] == 0 ? 4 : 2;
        if (!g[i] || ((uintptr_t)g[i] & (es - 1))) return bad("null or misaligned gradient");
        ranges.emplace_back((uintptr_t)g[i], (uintptr_t)g[i] + (size_t)counts[i] * es);
        Entry e = {g[i], nullptr, nullptr, nullptr, counts[i], 0, types[i], i, 0, 0};
        if (A.adam) {
            e.p = p[i]; e.m = m[i]; e.v = v[i];
            for (float* q : {e.p, e.m, e.v}) {
                if (!q || ((uintptr_t)q & 3)) return bad("null or misaligned parameter or moment");
                ranges.emplace_back((uintptr_t)q, (uintptr_t)q + (size_t)counts[i] * 4);
            }
        }
        tab.push_back(e);
        total += counts[i];
    }
    if (overlap(ranges)) return bad("tensors share memory (the same tensor twice?)");
    int dev = 0, nsm = 148;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&nsm, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) { set_error((int)e, who, cudaGetErrorString(e)); return -1; }
    // chunks that give every resident block one, within bounds: a longer one keeps more loads in flight
    const long long per = (total / ((long long)nsm * NORM_CTAS) + 1023) & ~1023ll;
    A.ch = (int)std::min<long long>(CH_BIG, std::max<long long>(CH_SMALL, per));
    long long c0 = 0;
    for (Entry& q : tab) { q.chunk0 = c0; c0 += (q.n + CH_SMALL - 1) / CH_SMALL; }
    const bool small = c0 <= CL * R && (A.adam ? cluster_fits<true>(dev) : cluster_fits<false>(dev));
    if (!small) {
        c0 = 0;
        for (Entry& q : tab) {
            const long long size = A.adam || q.type == 0 ? 4 : 2;
            q.head = (int)std::min<long long>(q.n, (long long)(-(uintptr_t)(A.adam ? (void*)q.p : q.g) & 127) / size);
            q.chunk0 = c0;
            c0 += std::max(1ll, (q.n - q.head + A.ch - 1) / A.ch);
        }
    }
    A.chunks = c0;
    A.n = (int)tab.size();
    A.steps = steps;
    A.part = (double*)ws;
    A.bias = (float2*)(A.part + MAX_PARTS + 1);
    Table<TAB> T = {};
    A.table = nullptr;
    if (A.n <= TAB) {
        for (int i = 0; i < A.n; ++i) T.e[i] = tab[i];
    } else {
        Entry* dst = (Entry*)(((uintptr_t)(A.bias + n) + 15) & ~(uintptr_t)15);
        static thread_local Table<TAB_BIG> B;
        for (int i = 0; i < A.n; i += TAB_BIG) {
            const int cnt = std::min(TAB_BIG, A.n - i);
            for (int k = 0; k < cnt; ++k) B.e[k] = tab[i + k];
            e = go(1, k_table, (cnt + 15) / 16, 32, st, B, cnt, dst + i);
            if (e != cudaSuccess) break;
        }
        A.table = dst;
    }
    if (e == cudaSuccess && small) {
        e = A.adam ? go(CL, k_small<true>, CL, CL_THREADS, st, A, T) : go(CL, k_small<false>, CL, CL_THREADS, st, A, T);
    } else if (e == cudaSuccess) {
        if (A.chunks >= (1ll << 31)) return bad("too many numbers");
        const int grid = (int)std::max(1ll, std::min<long long>(A.chunks, std::min(nsm * NORM_CTAS, MAX_PARTS)));
        A.nparts = grid;
        e = go(1, k_norm, grid, THREADS, st, A, T);
        if (A.chunks <= grid) {
            if (e == cudaSuccess) e = A.adam ? go(1, k_apply<true, true>, grid, THREADS, st, A, T) : go(1, k_apply<true, false>, grid, THREADS, st, A, T);
        } else {
            if (e == cudaSuccess) e = go(1, k_total, 1, 1024, st, A);
            const int all = (int)A.chunks;
            if (e == cudaSuccess) e = A.adam ? go(1, k_apply<false, true>, all, THREADS, st, A, T) : go(1, k_apply<false, false>, all, THREADS, st, A, T);
        }
    }
    if (e != cudaSuccess) { set_error((int)e, who, cudaGetErrorString(e)); return -1; }
    return 0;
}

}  // namespace g1opt

extern "C" {

long long g1_opt_workspace(int n) { return n < 0 ? 0 : (long long)g1opt::ws_bytes(n); }

int g1_clip_grad_norm(int n, void* const* grads, const int* types, const long long* counts, double max_norm, float* norm,
                      void* ws, long long ws_size, void* stream) {
    try {
        g1opt::Args A = {};
        A.max_norm = max_norm;
        A.norm = norm;
        return g1opt::run("g1_clip_grad_norm", n, grads, types, nullptr, nullptr, nullptr, counts, nullptr, A, ws, ws_size,
                          (cudaStream_t)stream);
    } catch (const std::bad_alloc&) {
        set_error(-12, "g1_clip_grad_norm", "out of host memory");
        return -12;
    }
}

int g1_clip_adam(int n, void* const* grads, const int* types, float* const* p, float* const* m, float* const* v,
                 const long long* counts, long long* steps, double max_norm, double lr, const float* lr_dev, double beta1,
                 double beta2, double eps, double weight_decay, float* norm, void* ws, long long ws_size, void* stream) {
    if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0) || !(lr >= 0.0) ||
        !(weight_decay >= 0.0) || ((uintptr_t)lr_dev & 3)) {
        set_error(-22, "g1_clip_adam", "betas must lie in [0, 1); lr, eps and weight_decay must be >= 0");
        return -22;
    }
    try {
        g1opt::Args A = {};
        A.max_norm = max_norm;
        A.adam = 1;
        A.b1d = beta1; A.b2d = beta2;
        A.omb1 = (float)(1.0 - beta1);
        A.b2 = (float)beta2;
        A.omb2 = (float)(1.0 - beta2);
        A.eps = (float)eps; A.lr = (float)lr; A.wd = (float)weight_decay;
        A.lr_dev = lr_dev;
        A.norm = norm;
        return g1opt::run("g1_clip_adam", n, grads, types, p, m, v, counts, steps, A, ws, ws_size, (cudaStream_t)stream);
    } catch (const std::bad_alloc&) {
        set_error(-12, "g1_clip_adam", "out of host memory");
        return -12;
    }
}

}  // extern "C"
