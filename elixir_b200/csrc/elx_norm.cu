// Part of the elixir_b200 CUDA library (C ABI: include/elixir_b200.h): layer norm, forward and backward.
//
//   mean = sum x / C,  rstd = 1 / sqrt(sum (x - mean)^2 / C + eps),  xhat = (x - mean) rstd,  y = xhat w + b
//   a = dy w,  dx = rstd (a - mean(a) - xhat mean(a xhat)),  dw = sum over rows dy xhat,  db = sum over rows dy
//
// Statistics, sums and the products that enter them are fp32; every output is rounded once.  A row is read once and
// stays in registers between the passes over it.
#include "elx_common.cuh"

using namespace elx;

namespace {

// The values of a piece are worked on in pairs (packed fp32 arithmetic: these kernels run short of issue slots before they
// run short of bandwidth), or one by one where a piece is one element.
template <int VEC>
struct Values {
    using E = float2;
    static constexpr int kN = VEC / 2;
    static __device__ __forceinline__ E all(float x) { return make_float2(x, x); }
    static __device__ __forceinline__ float sum(E x) { return x.x + x.y; }
};
template <>
struct Values<1> {
    using E = float;
    static constexpr int kN = 1;
    static __device__ __forceinline__ E all(float x) { return x; }
    static __device__ __forceinline__ float sum(E x) { return x; }
};

// VEC consecutive elements as they are held in memory: one 16-byte access (VEC = 8 of a 16-bit type, 4 of fp32), or one
// element, kept as fp32.
template <int DT, int VEC>
struct Piece {
    uint32_t w[4];
    __device__ __forceinline__ void zero() { w[0] = w[1] = w[2] = w[3] = 0; }
    __device__ __forceinline__ void load(const void* base, int64_t i) {
        const uint4 r = *reinterpret_cast<const uint4*>(static_cast<const typename Lp<DT>::T*>(base) + i);
        w[0] = r.x; w[1] = r.y; w[2] = r.z; w[3] = r.w;
    }
    __device__ __forceinline__ void get(float2 (&f)[VEC / 2]) const {
        if constexpr (DT == ELX_F32) {
            f[0] = make_float2(__uint_as_float(w[0]), __uint_as_float(w[1]));
            f[1] = make_float2(__uint_as_float(w[2]), __uint_as_float(w[3]));
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = Lp<DT>::unpack2(w[j]);
        }
    }
    __device__ __forceinline__ void put(const float2 (&f)[VEC / 2]) {
        if constexpr (DT == ELX_F32) {
            w[0] = __float_as_uint(f[0].x); w[1] = __float_as_uint(f[0].y);
            w[2] = __float_as_uint(f[1].x); w[3] = __float_as_uint(f[1].y);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = Lp<DT>::pack2(f[j].x, f[j].y);
        }
    }
    __device__ __forceinline__ void store(void* base, int64_t i) const {
        *reinterpret_cast<uint4*>(static_cast<typename Lp<DT>::T*>(base) + i) = make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <int DT>
struct Piece<DT, 1> {
    float x;
    __device__ __forceinline__ void zero() { x = 0.0f; }
    __device__ __forceinline__ void load(const void* base, int64_t i) {
        x = Lp<DT>::to_float(static_cast<const typename Lp<DT>::T*>(base)[i]);
    }
    __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = x; }
    __device__ __forceinline__ void put(const float (&f)[1]) { x = f[0]; }
    __device__ __forceinline__ void store(void* base, int64_t i) const {
        static_cast<typename Lp<DT>::T*>(base)[i] = Lp<DT>::from_float(x);
    }
};

template <int DT>
struct Wide {
    static constexpr int kVec = DT == ELX_F32 ? 4 : 8;
};

// Rows of a width that 16-byte pieces do not divide do not begin on 16-byte boundaries, but all rows r with the same
// (mis + r cols) mod V begin at one distance, `shift`, from one.  A thread that keeps to such rows keeps its columns: piece P
// of a row holds columns P V - shift + [0, V), those outside [0, cols) belonging to the neighbours.
struct Span {
    int c;         // first column of the piece
    bool any;      // some of its columns are the row's
    bool full;     // all of them are
};
template <int VEC>
__device__ __forceinline__ Span span_of(int piece, int shift, int cols) {
    Span s;
    s.c = piece * VEC - shift;
    s.any = s.c < cols && s.c + VEC > 0;
    s.full = s.c >= 0 && s.c + VEC <= cols;
    return s;
}
// Columns [c, c + V) of an array at any alignment, zero outside [0, cols): V loads that are on their way together.
template <int DT>
__device__ __forceinline__ uint4 load_columns(const void* base, int64_t at, int c, int cols) {
    constexpr int VEC = Wide<DT>::kVec;
    uint32_t x[VEC], w[4];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const int k = min(max(c + j, 0), cols - 1) - c;
        if constexpr (DT == ELX_F32) x[j] = static_cast<const uint32_t*>(base)[at + k];
        else x[j] = static_cast<const uint16_t*>(base)[at + k];
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j)
        if (c + j < 0 || c + j >= cols) x[j] = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (DT == ELX_F32) w[j] = x[j];
        else w[j] = x[2 * j] | (x[2 * j + 1] << 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <int DT>
__device__ __noinline__ void store_end(void* base, int64_t at, int c, int cols, uint4 r) {
    constexpr int VEC = Wide<DT>::kVec;
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        if (c + j < 0 || c + j >= cols) continue;
        if constexpr (DT == ELX_F32) static_cast<uint32_t*>(base)[at + j] = w[j];
        else static_cast<uint16_t*>(base)[at + j] = static_cast<uint16_t>(w[j / 2] >> (16 * (j & 1)));
    }
}
// A piece on its way, whatever of it is the row's; only one that reaches outside the array (of `total` elements) is read
// element by element.  trim() then zeroes the neighbours' elements, once the piece is needed.
template <int DT, int VEC>
__device__ __forceinline__ void load_span(Piece<DT, VEC>& p, const void* base, const Span& s, int64_t at, int cols, int64_t total) {
    if (!s.any) return;
    if (s.full || (at >= 0 && at + VEC <= total)) {
        p.load(base, at);
    } else {
        const uint4 r = load_columns<DT>(base, at, s.c, cols);
        p.w[0] = r.x; p.w[1] = r.y; p.w[2] = r.z; p.w[3] = r.w;
    }
}
template <int DT, int VEC>
__device__ __forceinline__ void trim(Piece<DT, VEC>& p, const Span& s, int cols) {
    if (s.full) return;
    constexpr int kPer = VEC / 4;
#pragma unroll
    for (int j = 0; j < VEC; ++j)
        if (s.c + j < 0 || s.c + j >= cols) p.w[j / kPer] &= kPer == 1 ? 0u : (j & 1) ? 0xFFFFu : 0xFFFF0000u;
}
// The parameters of a piece's columns: they lie at any distance from a boundary.
template <int DT, int VEC>
__device__ __forceinline__ void load_parameters(Piece<DT, VEC>& p, const void* base, const Span& s, int cols) {
    if (!s.any) return;
    const uint4 r = load_columns<DT>(base, s.c, s.c, cols);
    p.w[0] = r.x; p.w[1] = r.y; p.w[2] = r.z; p.w[3] = r.w;
}
template <int DT, int VEC>
__device__ __forceinline__ void store_span(const Piece<DT, VEC>& p, void* base, const Span& s, int64_t at, int cols) {
    if (s.full) p.store(base, at);
    else if (s.any) store_end<DT>(base, at, s.c, cols, make_uint4(p.w[0], p.w[1], p.w[2], p.w[3]));
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

// Sums of two values over a warp: half of the lanes take over one of them first, 6 exchanges instead of 10.  Lanes 0 to 15
// end up with the first sum, the others with the second.
__device__ __forceinline__ float warp_sum_pair(float a, float b) {
    const bool high = threadIdx.x & 16;
    float v = (high ? b : a) + __shfl_xor_sync(0xFFFFFFFFu, high ? a : b, 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

// Sums of N values over the threads of a block; every thread gets them.  s: N * 32 floats, not used by another sum
// between two barriers.
template <int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float* s) {
    const int warps = (blockDim.x + 31) >> 5, w = threadIdx.x >> 5;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) s[i * 32 + w] = v[i];
    __syncthreads();
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_sum(lane < warps ? s[i * 32 + lane] : 0.0f);
}

struct NormArgs {
    const void* x;
    const void* weight;
    const void* bias;
    const void* dy;
    void* out;          // y or dx
    float* mean;
    float* rstd;
    float* partial;     // backward: groups x 2 x cols
    int64_t rows;
    int cols;
    int groups;         // backward: how many blocks have a partial sum of their own
    int group_threads;  // threads that share a row
    int mis;            // elements from a 16-byte boundary to x's first one (and to every other array's of its shape)
    float eps;
};

// Threads per block that the registers of VPL pieces allow.
constexpr int max_threads(int vec, int vpl) {
    const int words = vec == 1 ? vpl : 4 * vpl;
    return words <= 16 ? 1024 : words <= 40 ? 512 : 256;
}

// One row per warp (ONE: several rows per block, no barrier) or per block.  The row is read once and stays in registers
// as it is held in memory; the mean comes first and the spread from the differences, so a large mean costs no digits.
// Bound by the bytes in flight: a warp has its whole row on the way before it adds the first element.  fp16 8192 x 1600
// 13.2 us (4.0 TB/s; both arrays fit the L2), 16384 x 2048 25.7 us (5.2 TB/s), 16384 x 4096 50 us (5.4 TB/s); one row 3.2 us.
template <int DT, int VEC, int VPL, bool ONE>
__global__ void __launch_bounds__(ONE ? 128 : max_threads(VEC, VPL)) norm_forward_kernel(const NormArgs a) {
    __shared__ float s_sum[ONE ? 1 : 2][32];
    const int t = ONE ? threadIdx.x & 31 : threadIdx.x, threads = ONE ? 32 : blockDim.x;
    const int64_t row = ONE ? static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    if (ONE && row >= a.rows) return;   // the whole warp
    Piece<DT, VEC> x[VPL];
    const int64_t base = row * a.cols;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const int c = (i * threads + t) * VEC;
        if (c < a.cols) x[i].load(a.x, base + c);
        else x[i].zero();
    }
    using V = Values<VEC>;
    using E = typename V::E;
    E acc = V::all(0.0f), f[V::kN];
    float sum[1];
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        x[i].get(f);
#pragma unroll
        for (int j = 0; j < V::kN; ++j) acc = add2(acc, f[j]);
    }
    sum[0] = V::sum(acc);
    if constexpr (ONE) sum[0] = warp_sum(sum[0]);
    else block_sum<1>(sum, s_sum[0]);
    const float mean = sum[0] / static_cast<float>(a.cols);
    acc = V::all(0.0f);
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        if ((i * threads + t) * VEC >= a.cols) continue;
        x[i].get(f);
#pragma unroll
        for (int j = 0; j < V::kN; ++j) {
            const E d = add2(f[j], V::all(-mean));
            acc = fma2(d, d, acc);
        }
    }
    sum[0] = V::sum(acc);
    if constexpr (ONE) sum[0] = warp_sum(sum[0]);
    else block_sum<1>(sum, s_sum[1]);
    const float rstd = 1.0f / sqrtf(sum[0] / static_cast<float>(a.cols) + a.eps);
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const int c = (i * threads + t) * VEC;
        if (c >= a.cols) continue;
        Piece<DT, VEC> pw, pb;
        E w[V::kN], b[V::kN];
        if (a.weight) {
            pw.load(a.weight, c);
            pw.get(w);
        }
        if (a.bias) {
            pb.load(a.bias, c);
            pb.get(b);
        }
        x[i].get(f);
#pragma unroll
        for (int j = 0; j < V::kN; ++j) {
            f[j] = mul2(add2(f[j], V::all(-mean)), V::all(rstd));
            if (a.weight) f[j] = mul2(f[j], w[j]);
            if (a.bias) f[j] = add2(f[j], b[j]);
        }
        x[i].put(f);
        x[i].store(a.out, base + c);
    }
    if (t == 0) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
    }
}

// Sum of one value over the threads of a group (a warp, or several with named barrier `id`); s: a float per warp.
__device__ __forceinline__ float group_sum(float v, float* s, int id, int threads, int t) {
    v = warp_sum(v);
    if (threads == 32) return v;
    if ((t & 31) == 0) s[t >> 5] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
    const int lane = t & 31;
    return warp_sum(lane < (threads >> 5) ? s[lane] : 0.0f);
}

// Rows of a width that 16-byte pieces do not divide.  Groups of threads walk over rows that all begin at one distance from
// a 16-byte boundary (their number is a multiple of V), so a thread's columns, weights and biases stay the same, and x and y
// move in 16-byte pieces but for the two ends of a row.  8192 x 1111: fp16 24 us (31 us with an access per element), and
// 8192 x 1601 fp32 37 us.  Bound by instructions: 31 per element, half of them for the ends of the rows; and row, next row,
// parameters and spans do not fit the registers: with two and four pieces per thread the 16-bit forms spill 180 to 212 bytes
// and read 228 to 240 back.
template <int DT, int VPL>
__global__ void __launch_bounds__(512, VPL > 2 ? 1 : 2) norm_forward_odd_kernel(const NormArgs a) {
    constexpr int VEC = Wide<DT>::kVec;
    __shared__ float s_sum[2][2][16][16];   // [row parity][which sum][group][warp]
    const int threads = a.group_threads, group = threadIdx.x / threads, t = threadIdx.x - group * threads;
    const int groups = blockDim.x / threads;
    const int64_t stride = static_cast<int64_t>(gridDim.x) * groups, total = a.rows * a.cols;
    int64_t row = static_cast<int64_t>(blockIdx.x) * groups + group;
    const int shift = static_cast<int>((a.mis + row * a.cols) % VEC);
    Piece<DT, VEC> x[VPL], next[VPL], w[VPL], b[VPL];
    Span span[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        span[i] = span_of<VEC>(i * threads + t, shift, a.cols);
        w[i].zero();
        b[i].zero();
        x[i].zero();
        next[i].zero();
        if (a.weight) load_parameters<DT, VEC>(w[i], a.weight, span[i], a.cols);
        if (a.bias) load_parameters<DT, VEC>(b[i], a.bias, span[i], a.cols);
        if (row < a.rows) load_span<DT, VEC>(x[i], a.x, span[i], row * a.cols + span[i].c, a.cols, total);
    }
    using V = Values<VEC>;
    const float inv = 1.0f / static_cast<float>(a.cols);
    for (int parity = 0; row < a.rows; row += stride, parity ^= 1) {
        if (row + stride < a.rows)
#pragma unroll
            for (int i = 0; i < VPL; ++i) load_span<DT, VEC>(next[i], a.x, span[i], (row + stride) * a.cols + span[i].c, a.cols, total);
        float2 acc = V::all(0.0f), f[V::kN];
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            trim<DT, VEC>(x[i], span[i], a.cols);
            x[i].get(f);
#pragma unroll
            for (int j = 0; j < V::kN; ++j) acc = add2(acc, f[j]);
        }
        const float mean = group_sum(V::sum(acc), s_sum[parity][0][group], 1 + group, threads, t) * inv;
        acc = V::all(0.0f);
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            if (!span[i].any) continue;
            x[i].get(f);
#pragma unroll
            for (int j = 0; j < V::kN; ++j) {
                float2 d = add2(f[j], V::all(-mean));
                if (!span[i].full) {   // the neighbours' places
                    const int c = span[i].c + 2 * j;
                    if (c < 0 || c >= a.cols) d.x = 0.0f;
                    if (c + 1 < 0 || c + 1 >= a.cols) d.y = 0.0f;
                }
                acc = fma2(d, d, acc);
            }
        }
        const float rstd = 1.0f / sqrtf(group_sum(V::sum(acc), s_sum[parity][1][group], 1 + group, threads, t) * inv + a.eps);
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            float2 fw[V::kN], fb[V::kN];
            x[i].get(f);
            w[i].get(fw);
            b[i].get(fb);
#pragma unroll
            for (int j = 0; j < V::kN; ++j) {
                f[j] = mul2(add2(f[j], V::all(-mean)), V::all(rstd));
                if (a.weight) f[j] = mul2(f[j], fw[j]);
                if (a.bias) f[j] = add2(f[j], fb[j]);
            }
            x[i].put(f);
            store_span<DT, VEC>(x[i], a.out, span[i], row * a.cols + span[i].c, a.cols);
            x[i] = next[i];
        }
        if (t == 0) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
    }
}

template <int DT>
__device__ __forceinline__ float load1(const void* base, int64_t i) {
    return Lp<DT>::to_float(static_cast<const typename Lp<DT>::T*>(base)[i]);
}
template <int DT>
__device__ __forceinline__ void store1(void* base, int64_t i, float x) {
    static_cast<typename Lp<DT>::T*>(base)[i] = Lp<DT>::from_float(x);
}

// Rows wider than the registers of a block: the row is read once per pass.
template <int DT>
__global__ void __launch_bounds__(1024) norm_forward_wide_kernel(const NormArgs a) {
    __shared__ float s_sum[2][32];
    const int64_t base = static_cast<int64_t>(blockIdx.x) * a.cols;
    float sum[1] = {0.0f};
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) sum[0] += load1<DT>(a.x, base + c);
    block_sum<1>(sum, s_sum[0]);
    const float mean = sum[0] / static_cast<float>(a.cols);
    sum[0] = 0.0f;
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
        const float d = load1<DT>(a.x, base + c) - mean;
        sum[0] = fmaf(d, d, sum[0]);
    }
    block_sum<1>(sum, s_sum[1]);
    const float rstd = 1.0f / sqrtf(sum[0] / static_cast<float>(a.cols) + a.eps);
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
        float y = (load1<DT>(a.x, base + c) - mean) * rstd;
        if (a.weight) y *= load1<DT>(a.weight, c);
        if (a.bias) y += load1<DT>(a.bias, c);
        store1<DT>(a.out, base + c, y);
    }
    if (threadIdx.x == 0) {
        a.mean[blockIdx.x] = mean;
        a.rstd[blockIdx.x] = rstd;
    }
}

// Several groups of threads per block, each walking over rows of its own (TPR threads per row, a thread VPL pieces of
// columns that stay the same from row to row).  The two column sums of a thread's columns live in registers; at the end
// the block's groups add theirs up in shared memory, in order, and one partial sum per block goes out.  A row takes one
// barrier among its threads; the next row's pieces are on their way meanwhile (NEXT).
// ODD: as norm_forward_odd_kernel, rows that 16-byte pieces do not divide; what a piece holds of a neighbouring row counts
// as zero gradients.
// With norm_columns_kernel, fp16: 8192 x 1600 23.5 us (3.3 TB/s), 16384 x 2048 41.8 us (4.8 TB/s), 16384 x 4096 78 us
// (5.2 TB/s); bound by what a row waits for: its loads, one barrier, its sums.  Rows of more than 1024 pieces (NEXT off) lose
// what is not on its way early: 4096 x 9216 113 us (2.0 TB/s); the 16-bit forms of these spill as well, 104 to 296 bytes (132 to
// 664 read back), and the odd ones of narrower rows up to 32.
// VPL 1 up to 96 pieces: 32768 x 768 fp16 37 us against 39 with two per thread, 65536 x 256 28.6 us against 31.4 in 512 threads;
// wider rows lose more by another warp's part of each row's sums (16384 x 1600 40 us with two per thread, 47 with one, 42 with
// three).
constexpr int backward_threads(int vpl) { return vpl == 1 ? 768 : 512; }
template <int DT, int VEC, int VPL, bool NEXT, bool ODD>
__global__ void __launch_bounds__(backward_threads(VPL), 1) norm_backward_kernel(const NormArgs a) {
    extern __shared__ float s_cols[];                 // 2 x cols, where there are several groups
    __shared__ float2 s_sum[2][24][16];               // [row parity][group][warp]
    const int threads = a.group_threads, group = threadIdx.x / threads, t = threadIdx.x - group * threads;
    const int groups = blockDim.x / threads, warps = threads >> 5, warp = t >> 5;
    using V = Values<VEC>;
    using E = typename V::E;
    // KEPT (fp32): differences and products of a row's first half stay in registers for the second, and the next row is asked
    // for in between.  Else both are formed again from the row as it is held, and the next row is asked for at once: 16-bit
    // rows hold twice the elements in those registers (8192 x 1600: fp32 37 us against 49, fp16 24.5 us against 24.8;
    // 16384 x 4096 bf16 107 us against 79).
    constexpr bool KEPT = NEXT && DT == ELX_F32, EARLY = NEXT && !KEPT;
    Piece<DT, VEC> w[NEXT ? VPL : 1], x[VPL], dy[VPL], nx[EARLY ? VPL : 1], ndy[EARLY ? VPL : 1];
    E dw[VPL][V::kN], db[VPL][V::kN];
    const int64_t stride = static_cast<int64_t>(gridDim.x) * groups, total = a.rows * a.cols;
    int64_t row = static_cast<int64_t>(blockIdx.x) * groups + group;
    const int shift = ODD ? static_cast<int>((a.mis + row * a.cols) % VEC) : 0;
    Span span[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        if constexpr (ODD) {
            span[i] = span_of<VEC>(i * threads + t, shift, a.cols);
        } else {
            span[i].c = (i * threads + t) * VEC;
            span[i].any = span[i].full = span[i].c < a.cols;
        }
        x[i].zero();
        dy[i].zero();
        if constexpr (EARLY) {
            nx[i].zero();
            ndy[i].zero();
        }
        if constexpr (NEXT) {
            w[i].zero();
            if constexpr (ODD) {
                if (a.weight) load_parameters<DT, VEC>(w[i], a.weight, span[i], a.cols);
            } else {
                if (a.weight && span[i].any) w[i].load(a.weight, span[i].c);
            }
        }
#pragma unroll
        for (int j = 0; j < V::kN; ++j) dw[i][j] = db[i][j] = V::all(0.0f);
    }
    const float inv = 1.0f / static_cast<float>(a.cols);
    float mean = 0.0f, rstd = 0.0f;
    auto fetch = [&](int64_t r, Piece<DT, VEC>* px, Piece<DT, VEC>* pdy, float& m, float& s) {
        m = a.mean[r];
        s = a.rstd[r];
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int64_t at = r * a.cols + span[i].c;
            if constexpr (ODD) {
                load_span<DT, VEC>(px[i], a.x, span[i], at, a.cols, total);
                load_span<DT, VEC>(pdy[i], a.dy, span[i], at, a.cols, total);
            } else if (span[i].any) {
                px[i].load(a.x, at);
                pdy[i].load(a.dy, at);
            }
        }
    };
    auto weights = [&](int i, E (&f)[V::kN]) {   // kept in registers, or (wide rows) read again from the cache
        if constexpr (NEXT) {
            w[i].get(f);
        } else if (a.weight) {
            Piece<DT, VEC> p;
            p.zero();
            if constexpr (ODD) load_parameters<DT, VEC>(p, a.weight, span[i], a.cols);
            else p.load(a.weight, span[i].c);
            p.get(f);
        }
    };
    if (NEXT && row < a.rows) fetch(row, x, dy, mean, rstd);
    float next_mean = 0.0f, next_rstd = 0.0f;
    E d[KEPT ? VPL : 1][V::kN], g[KEPT ? VPL : 1][V::kN];
    for (int parity = 0; row < a.rows; row += stride, parity ^= 1) {
        if constexpr (!NEXT) fetch(row, x, dy, mean, rstd);
        if constexpr (EARLY) {
            if (row + stride < a.rows) fetch(row + stride, nx, ndy, next_mean, next_rstd);
        }
        const float now_rstd = rstd;
        const E scale = V::all(rstd), minus = V::all(-mean);
        E sum0 = V::all(0.0f), sum1 = V::all(0.0f), fx[V::kN], fd[V::kN], fw[V::kN];
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            if (!span[i].any) continue;
            if constexpr (ODD) {
                trim<DT, VEC>(x[i], span[i], a.cols);
                trim<DT, VEC>(dy[i], span[i], a.cols);
            }
            x[i].get(fx);
            dy[i].get(fd);
            weights(i, fw);
#pragma unroll
            for (int j = 0; j < V::kN; ++j) {
                const E diff = add2(fx[j], minus), xhat = mul2(diff, scale);
                dw[i][j] = fma2(fd[j], xhat, dw[i][j]);
                db[i][j] = add2(db[i][j], fd[j]);
                const E prod = a.weight ? mul2(fd[j], fw[j]) : fd[j];
                sum0 = add2(sum0, prod);
                sum1 = fma2(prod, xhat, sum1);
                if constexpr (KEPT) {
                    d[i][j] = diff;
                    g[i][j] = prod;
                }
            }
        }
        if constexpr (KEPT) {
            if (row + stride < a.rows) fetch(row + stride, x, dy, mean, rstd);
        }
        const float pair = warp_sum_pair(V::sum(sum0), V::sum(sum1));
        float2 sum;
        if (warps > 1) {
            // one barrier per row: the next row writes the other half, and the row after it only past the next barrier
            if ((t & 15) == 0) reinterpret_cast<float*>(&s_sum[parity][group][warp])[(t >> 4) & 1] = pair;
            asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(threads) : "memory");
            sum = s_sum[parity][group][0];
            for (int j = 1; j < warps; ++j) {
                const float2 o = s_sum[parity][group][j];
                sum.x += o.x;
                sum.y += o.y;
            }
        } else {
            sum.x = __shfl_sync(0xFFFFFFFFu, pair, 0);
            sum.y = __shfl_sync(0xFFFFFFFFu, pair, 16);
        }
        // dx = rstd (g - m0 - (x - mean) rstd m1): exactly zero where there is nothing to spread over
        const E m0 = V::all(-(sum.x * inv)), m1 = V::all(-(sum.y * inv) * now_rstd);
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            if (!span[i].any) continue;
            if constexpr (!KEPT) {
                x[i].get(fx);
                dy[i].get(fd);
                weights(i, fw);
            }
#pragma unroll
            for (int j = 0; j < V::kN; ++j) {
                if constexpr (KEPT) {
                    fd[j] = mul2(scale, fma2(d[i][j], m1, add2(g[i][j], m0)));
                } else {
                    const E prod = a.weight ? mul2(fd[j], fw[j]) : fd[j];
                    fd[j] = mul2(scale, fma2(add2(fx[j], minus), m1, add2(prod, m0)));
                }
            }
            Piece<DT, VEC> out;
            out.put(fd);
            if constexpr (ODD) store_span<DT, VEC>(out, a.out, span[i], row * a.cols + span[i].c, a.cols);
            else out.store(a.out, row * a.cols + span[i].c);
        }
        if constexpr (EARLY) {
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                x[i] = nx[i];
                dy[i] = ndy[i];
            }
            mean = next_mean;
            rstd = next_rstd;
        }
    }
    next_may_start();
    if (!a.partial) return;
    float* const part = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.cols;
    for (int g = 0; g < groups; ++g) {
        if (g == group) {
            float* const to = g == groups - 1 ? part : s_cols;
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                if (!span[i].any) continue;
                const float* const dwf = reinterpret_cast<const float*>(dw[i]);
                const float* const dbf = reinterpret_cast<const float*>(db[i]);
                if constexpr (!ODD && VEC > 1) {
#pragma unroll
                    for (int j = 0; j < VEC; j += 4) {
#pragma unroll
                        for (int which = 0; which < 2; ++which) {
                            const float* const f = which ? dbf : dwf;
                            const int c = which * a.cols + span[i].c + j;
                            float4 v = make_float4(f[j], f[j + 1], f[j + 2], f[j + 3]);
                            if (g) {
                                const float4 o = *reinterpret_cast<const float4*>(s_cols + c);
                                v = make_float4(o.x + v.x, o.y + v.y, o.z + v.z, o.w + v.w);
                            }
                            *reinterpret_cast<float4*>(to + c) = v;
                        }
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const int c = span[i].c + j;
                        if (ODD && (c < 0 || c >= a.cols)) continue;
                        to[c] = (g ? s_cols[c] : 0.0f) + dwf[j];
                        to[a.cols + c] = (g ? s_cols[a.cols + c] : 0.0f) + dbf[j];
                    }
                }
            }
        }
        if (groups > 1) __syncthreads();
    }
}

// Wide rows: dx row by row, and the column sums in a pass of their own, an access per element (1000 x 40000 fp16: 228 us).
// fp32 rows come here from 8196 columns on: 4096 x 9216 215 us, where a pass over the bytes takes 70.
template <int DT>
__global__ void __launch_bounds__(1024) norm_backward_wide_kernel(const NormArgs a) {
    __shared__ float s_sum[2 * 32];
    const int64_t row = blockIdx.x, base = row * a.cols;
    const float mean = a.mean[row], rstd = a.rstd[row], inv = 1.0f / static_cast<float>(a.cols);
    float sum[2] = {0.0f, 0.0f};
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
        const float g = load1<DT>(a.dy, base + c) * (a.weight ? load1<DT>(a.weight, c) : 1.0f);
        sum[0] += g;
        sum[1] = fmaf(g, (load1<DT>(a.x, base + c) - mean) * rstd, sum[1]);
    }
    block_sum<2>(sum, s_sum);
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
        const float g = load1<DT>(a.dy, base + c) * (a.weight ? load1<DT>(a.weight, c) : 1.0f);
        const float xhat = (load1<DT>(a.x, base + c) - mean) * rstd;
        store1<DT>(a.out, base + c, rstd * (g - sum[0] * inv - xhat * (sum[1] * inv)));
    }
}
template <int DT>
__global__ void __launch_bounds__(256) norm_columns_wide_kernel(const NormArgs a) {
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= a.cols) return;
    float dw = 0.0f, db = 0.0f;
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float dy = load1<DT>(a.dy, row * a.cols + c);
        dw = fmaf(dy, (load1<DT>(a.x, row * a.cols + c) - a.mean[row]) * a.rstd[row], dw);
        db += dy;
    }
    a.partial[static_cast<int64_t>(blockIdx.y) * 2 * a.cols + c] = dw;
    a.partial[(static_cast<int64_t>(blockIdx.y) * 2 + 1) * a.cols + c] = db;
}

// Sum of the partial column sums, in a fixed order: 32 columns x 32 slices of the groups per block.
template <int DT>
__global__ void __launch_bounds__(1024) norm_columns_kernel(const float* __restrict__ partial, int groups, int cols, void* dweight,
                                                            void* dbias) {
    __shared__ float s[2][32][33];
    const int c = blockIdx.x * 32 + threadIdx.x;
    float dw = 0.0f, db = 0.0f;
    after_previous();
    if (c < cols) {
        for (int g = threadIdx.y; g < groups; g += 32) {
            dw += partial[static_cast<int64_t>(g) * 2 * cols + c];
            db += partial[(static_cast<int64_t>(g) * 2 + 1) * cols + c];
        }
    }
    s[0][threadIdx.y][threadIdx.x] = dw;
    s[1][threadIdx.y][threadIdx.x] = db;
    __syncthreads();
    if (threadIdx.y >= 2 || c >= cols) return;
    void* const out = threadIdx.y == 0 ? dweight : dbias;
    if (!out) return;
    float t = 0.0f;
    for (int j = 0; j < 32; ++j) t += s[threadIdx.y][j][threadIdx.x];
    static_cast<typename Lp<DT>::T*>(out)[c] = Lp<DT>::from_float(t);
}

int round32(int n) { return (n + 31) / 32 * 32; }

template <int DT, int VEC, int VPL, bool ONE>
int launch_forward(const NormArgs& a, int warps, cudaStream_t s) {
    const int64_t grid = ONE ? (a.rows + 3) / 4 : a.rows;
    if (grid > 0x7FFFFFFF || (!ONE && 32 * warps > max_threads(VEC, VPL))) return ELX_ERR_CAPACITY;
    norm_forward_kernel<DT, VEC, VPL, ONE><<<static_cast<unsigned>(grid), ONE ? 128 : 32 * warps, 0, s>>>(a);
    return record_cuda(cudaGetLastError());
}

// Warps per row, by its width alone, so that a row's result does not depend on how many rows the call has: one, where the
// row fits a warp's registers in few pieces per lane, else as many as give each lane four (16, of one element), else 16 warps
// of as many as their registers hold.  Measured (GB/s of x and y, fp16): 8192 x 1600 in one warp 3740, in two 3460;
// 16384 x 4096 in one 3090, two 4070, four 5160, eight 3740.  On both sides of seven pieces, fp16: 32768 x 1792 (seven) 49 us
// in one warp, 53 us in two; 8192 x 1800 (eight) 22.3 us in one, 20.6 us in two, though 32768 rows of it take 52.5 and 53.6 us.
// 0: no such kernel.
template <int VEC>
int forward_warps(int pieces) {
    constexpr int kAlone = VEC == 1 ? 40 : 7, kEach = VEC == 1 ? 16 : 4, kMost = VEC == 1 ? 40 : 10;
    if (pieces <= 32 * kAlone) return 1;
    const int warps = (pieces + 32 * kEach - 1) / (32 * kEach);
    return warps <= 32 ? warps : pieces <= 32 * 16 * kMost ? 16 : 0;
}

// Blocks of a kernel whose groups of threads walk over rows: one per SM of a B200 at most, whatever the device, so that the
// order of sums depends on the sizes alone.  `whole`: groups in all have to be a multiple of this (rows of an odd width).
int row_blocks(int64_t rows, int per_block, int whole) {
    if (rows >= 144) return 148 * per_block % whole ? 144 : rows < 148 ? 144 : 148;
    return static_cast<int>(whole > 1 ? (rows + 7) / 8 * 8 : rows);
}
constexpr int kMaxBlocks = 148;

template <int DT, int VPL>
int launch_forward_odd(NormArgs a, cudaStream_t s) {
    constexpr int V = Wide<DT>::kVec;
    const int pieces = (a.cols + 2 * V - 2) / V;
    a.group_threads = round32((pieces + VPL - 1) / VPL);
    int per_block = 512 / a.group_threads;
    if (per_block > 15 && a.group_threads > 32) per_block = 15;   // named barriers
    const int each = VPL > 2 ? 1 : 2, blocks = each * row_blocks((a.rows + per_block * each - 1) / (per_block * each), per_block, V);
    norm_forward_odd_kernel<DT, VPL><<<blocks, per_block * a.group_threads, 0, s>>>(a);
    return record_cuda(cudaGetLastError());
}

// wide_ok: every row of every array begins on a 16-byte boundary.  same_mis: x, y (and dy) begin at one distance from one.
template <int DT>
int forward_dt(const NormArgs& a, bool wide_ok, bool same_mis, cudaStream_t s) {
    constexpr int V = Wide<DT>::kVec;
    if (!wide_ok && same_mis && a.cols >= 4 * V) {
        const int pieces = (a.cols + 2 * V - 2) / V;
        if (pieces <= 32) return launch_forward_odd<DT, 1>(a, s);
        if (pieces <= 512) return launch_forward_odd<DT, 2>(a, s);
        if (pieces <= 2048) return launch_forward_odd<DT, 4>(a, s);
    }
    const int warps = wide_ok ? forward_warps<V>(a.cols / V) : forward_warps<1>(a.cols);
    const int each = warps ? ((wide_ok ? a.cols / V : a.cols) + 32 * warps - 1) / (32 * warps) : 0;   // pieces per lane
    if (wide_ok && warps == 1) {
        switch (each) {
            case 1: return launch_forward<DT, V, 1, true>(a, warps, s);
            case 2: return launch_forward<DT, V, 2, true>(a, warps, s);
            case 3: return launch_forward<DT, V, 3, true>(a, warps, s);
            case 4: return launch_forward<DT, V, 4, true>(a, warps, s);
            case 5: return launch_forward<DT, V, 5, true>(a, warps, s);
            case 6: return launch_forward<DT, V, 6, true>(a, warps, s);
            case 7: return launch_forward<DT, V, 7, true>(a, warps, s);
        }
    } else if (wide_ok && warps) {
        if (each <= 3) return launch_forward<DT, V, 3, false>(a, warps, s);
        if (each == 4) return launch_forward<DT, V, 4, false>(a, warps, s);
        return launch_forward<DT, V, 10, false>(a, warps, s);
    } else if (warps == 1) {
        if (each == 1) return launch_forward<DT, 1, 1, true>(a, warps, s);
        if (each == 2) return launch_forward<DT, 1, 2, true>(a, warps, s);
        if (each <= 4) return launch_forward<DT, 1, 4, true>(a, warps, s);
        if (each <= 8) return launch_forward<DT, 1, 8, true>(a, warps, s);
        if (each <= 16) return launch_forward<DT, 1, 16, true>(a, warps, s);
        if (each <= 24) return launch_forward<DT, 1, 24, true>(a, warps, s);
        if (each <= 32) return launch_forward<DT, 1, 32, true>(a, warps, s);
        return launch_forward<DT, 1, 40, true>(a, warps, s);
    } else if (warps) {
        if (each <= 16) return launch_forward<DT, 1, 16, false>(a, warps, s);
        return launch_forward<DT, 1, 40, false>(a, warps, s);
    }
    if (a.rows > 0x7FFFFFFF) return ELX_ERR_CAPACITY;
    norm_forward_wide_kernel<DT><<<static_cast<unsigned>(a.rows), 1024, 0, s>>>(a);
    return record_cuda(cudaGetLastError());
}

template <int DT, int VEC, int VPL, bool NEXT, bool ODD>
int launch_backward(NormArgs& a, cudaStream_t s) {
    const int pieces = ODD ? (a.cols + 2 * VEC - 2) / VEC : (a.cols + VEC - 1) / VEC;
    a.group_threads = round32((pieces + VPL - 1) / VPL);
    int per_block = backward_threads(VPL) / a.group_threads;
    if (per_block > 15 && a.group_threads > 32) per_block = 15;   // named barriers
    while (per_block > 1 && a.rows < 148 * (per_block - 1)) --per_block;   // few rows: more blocks rather than fuller ones
    a.groups = row_blocks((a.rows + per_block - 1) / per_block, per_block, ODD ? VEC : 1);
    const int smem = per_block > 1 ? 2 * a.cols * 4 : 0;
    if (smem > 46 * 1024) return ELX_ERR_CAPACITY;   // cannot be: two groups have at most 8 x 512 columns
    norm_backward_kernel<DT, VEC, VPL, NEXT, ODD><<<a.groups, per_block * a.group_threads, smem, s>>>(a);
    return record_cuda(cudaGetLastError());
}

template <int DT>
int backward_dt(NormArgs& a, bool wide_ok, bool same_mis, void* dweight, void* dbias, cudaStream_t s) {
    constexpr int V = Wide<DT>::kVec;
    int rc = 1;
    if (wide_ok) {
        const int vecs = a.cols / V;
        if (vecs <= 96) rc = launch_backward<DT, V, 1, true, false>(a, s);
        else if (vecs <= 1024) rc = launch_backward<DT, V, 2, true, false>(a, s);
        else if (vecs <= 2048) rc = launch_backward<DT, V, 4, false, false>(a, s);
    } else if (same_mis && a.cols >= 4 * V) {
        const int pieces = (a.cols + 2 * V - 2) / V;
        if (pieces <= 96) rc = launch_backward<DT, V, 1, true, true>(a, s);
        else if (pieces <= 1024) rc = launch_backward<DT, V, 2, true, true>(a, s);
        else if (pieces <= 2048) rc = launch_backward<DT, V, 4, false, true>(a, s);
    } else {
        if (a.cols <= 64) rc = launch_backward<DT, 1, 2, true, false>(a, s);
        else if (a.cols <= 4096) rc = launch_backward<DT, 1, 8, true, false>(a, s);
    }
    if (rc == 1) {
        if (a.rows > 0x7FFFFFFF) return ELX_ERR_CAPACITY;
        norm_backward_wide_kernel<DT><<<static_cast<unsigned>(a.rows), 1024, 0, s>>>(a);
        rc = record_cuda(cudaGetLastError());
        if (rc == ELX_OK && a.partial) {
            a.groups = row_blocks(a.rows, 1, 1);
            norm_columns_wide_kernel<DT><<<dim3((a.cols + 255) / 256, a.groups), 256, 0, s>>>(a);
            rc = record_cuda(cudaGetLastError());
        }
    }
    if (rc != ELX_OK || !a.partial) return rc;
    const cudaError_t e = launch_next(norm_columns_kernel<DT>, dim3((a.cols + 31) / 32), dim3(32, 32), s, a.partial, a.groups, a.cols,
                                      dweight, dbias);
    if (e != cudaSuccess) (void)cudaGetLastError();
    return record_cuda(e);
}

// Elements from the last 16-byte boundary to p.
int misplaced(const void* p, int size) { return static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15u) / size); }

}  // namespace

extern "C" {

int elx_layer_norm_forward(const void* x, const void* weight, const void* bias, int dtype, int64_t rows, int64_t cols,
                           float eps, void* y, float* mean, float* rstd, void* stream) {
    if (rows != 0 && (!x || !y || !mean || !rstd)) return ELX_ERR_NULL;
    if (!dtype_ok(dtype)) return ELX_ERR_DTYPE;
    if (rows < 0 || cols <= 0) return ELX_ERR_SIZE;
    if (cols > ELX_NORM_MAX_COLS) return ELX_ERR_CAPACITY;
    const int size = dtype_bytes(dtype);
    if (!aligned(x, size) || !aligned(y, size) || (weight && !aligned(weight, size)) || (bias && !aligned(bias, size)) ||
        !aligned(mean, 4) || !aligned(rstd, 4))
        return ELX_ERR_ALIGN;
    if (!(eps >= 0.0f)) return ELX_ERR_ARG;
    if (rows == 0) return ELX_OK;
    NormArgs a = {};
    a.x = x;
    a.weight = weight;
    a.bias = bias;
    a.out = y;
    a.mean = mean;
    a.rstd = rstd;
    a.rows = rows;
    a.cols = static_cast<int>(cols);
    a.eps = eps;
    // 16-byte accesses need every row of every array on a 16-byte boundary
    const bool wide_ok = cols * size % 16 == 0 && aligned(x, 16) && aligned(y, 16) && aligned(weight, 16) && aligned(bias, 16);
    a.mis = misplaced(x, size);
    const bool same_mis = a.mis == misplaced(y, size);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case ELX_F16: return forward_dt<ELX_F16>(a, wide_ok, same_mis, s);
        case ELX_BF16: return forward_dt<ELX_BF16>(a, wide_ok, same_mis, s);
    }
    return forward_dt<ELX_F32>(a, wide_ok, same_mis, s);
}

int64_t elx_layer_norm_backward_workspace(int64_t rows, int64_t cols) {
    if (rows < 0 || cols <= 0) return ELX_ERR_SIZE;
    return (rows < kMaxBlocks ? (rows + 7) / 8 * 8 : kMaxBlocks) * 2 * cols * 4;   // a partial sum per block at most
}

int elx_layer_norm_backward(const void* dy, const void* x, const void* weight, const float* mean, const float* rstd, int dtype,
                            int64_t rows, int64_t cols, void* dx, void* dweight, void* dbias, void* workspace,
                            int64_t workspace_bytes, void* stream) {
    if (rows != 0 && (!dy || !x || !mean || !rstd || !dx)) return ELX_ERR_NULL;
    if (!dtype_ok(dtype)) return ELX_ERR_DTYPE;
    if (rows < 0 || cols <= 0) return ELX_ERR_SIZE;
    if (cols > ELX_NORM_MAX_COLS) return ELX_ERR_CAPACITY;
    const int size = dtype_bytes(dtype);
    if (!aligned(dy, size) || !aligned(x, size) || !aligned(dx, size) || (weight && !aligned(weight, size)) ||
        (dweight && !aligned(dweight, size)) || (dbias && !aligned(dbias, size)) || !aligned(mean, 4) || !aligned(rstd, 4))
        return ELX_ERR_ALIGN;
    const bool sums = dweight || dbias;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (rows == 0) {   // the sums over no rows
        if (dweight && cudaMemsetAsync(dweight, 0, cols * size, s) != cudaSuccess) return record_cuda(cudaGetLastError());
        if (dbias && cudaMemsetAsync(dbias, 0, cols * size, s) != cudaSuccess) return record_cuda(cudaGetLastError());
        return ELX_OK;
    }
    if (sums) {
        if (!workspace) return ELX_ERR_NULL;
        if (!aligned(workspace, 16)) return ELX_ERR_ALIGN;
        if (workspace_bytes < elx_layer_norm_backward_workspace(rows, cols)) return ELX_ERR_CAPACITY;
    }
    NormArgs a = {};
    a.dy = dy;
    a.x = x;
    a.weight = weight;
    a.mean = const_cast<float*>(mean);
    a.rstd = const_cast<float*>(rstd);
    a.out = dx;
    a.partial = sums ? static_cast<float*>(workspace) : nullptr;
    a.rows = rows;
    a.cols = static_cast<int>(cols);
    a.mis = misplaced(x, size);
    const bool same_mis = a.mis == misplaced(dy, size) && a.mis == misplaced(dx, size);
    const bool wide_ok = cols * size % 16 == 0 && aligned(x, 16) && aligned(dy, 16) && aligned(dx, 16) && aligned(weight, 16);
    switch (dtype) {
        case ELX_F16: return backward_dt<ELX_F16>(a, wide_ok, same_mis, dweight, dbias, s);
        case ELX_BF16: return backward_dt<ELX_BF16>(a, wide_ok, same_mis, dweight, dbias, s);
    }
    return backward_dt<ELX_F32>(a, wide_ok, same_mis, dweight, dbias, s);
}

}  // extern "C"
