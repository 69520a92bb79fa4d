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

// VEC consecutive elements as fp32: one 16-byte access (VEC = 8 of a 16-bit type, 4 of fp32) or one element.
template <int DT, int VEC>
__device__ __forceinline__ void load_vec(const void* base, int64_t i, float (&f)[VEC]) {
    using T = typename Lp<DT>::T;
    if constexpr (VEC == 1) {
        f[0] = Lp<DT>::to_float(static_cast<const T*>(base)[i]);
    } else {
        const uint4 r = *reinterpret_cast<const uint4*>(static_cast<const T*>(base) + i);
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
        if constexpr (DT == ELX_F32) {
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = __uint_as_float(w[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 p = Lp<DT>::unpack2(w[j]);
                f[2 * j] = p.x;
                f[2 * j + 1] = p.y;
            }
        }
    }
}
template <int DT, int VEC>
__device__ __forceinline__ void store_vec(void* base, int64_t i, const float (&f)[VEC]) {
    using T = typename Lp<DT>::T;
    if constexpr (VEC == 1) {
        static_cast<T*>(base)[i] = Lp<DT>::from_float(f[0]);
    } else {
        uint4 r;
        if constexpr (DT == ELX_F32) {
            r = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
        } else {
            r = make_uint4(Lp<DT>::pack2(f[0], f[1]), Lp<DT>::pack2(f[2], f[3]), Lp<DT>::pack2(f[4], f[5]),
                           Lp<DT>::pack2(f[6], f[7]));
        }
        *reinterpret_cast<uint4*>(static_cast<T*>(base) + i) = r;
    }
}

template <int DT>
struct Wide {
    static constexpr int kVec = DT == ELX_F32 ? 4 : 8;
};

// Sums of N values over the blockDim.x threads of each row (blockDim.y rows per block); every thread gets them.
// s: N * 32 floats per row.  All threads of the block call it; `s` may be reused after the next call returns.
template <int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* s) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xFFFFFFFFu, v[i], o);
    if (blockDim.x == 32) return;
    const int warps = blockDim.x >> 5, w = threadIdx.x >> 5;
    s += threadIdx.y * (N * 32);
    __syncthreads();
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) s[i * 32 + w] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float t = 0.0f;
        for (int j = 0; j < warps; ++j) t += s[i * 32 + j];
        v[i] = t;
    }
}

constexpr int kMaxRowsPerBlock = 8;

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
    int groups;         // backward: how many groups of rows have a partial sum of their own
    float eps;
};

template <int DT, int VEC, int VPT>
__global__ void __launch_bounds__(1024) norm_forward_kernel(const NormArgs a) {
    __shared__ float s_sum[kMaxRowsPerBlock * 32];
    const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
    const bool live = row < a.rows;
    float x[VPT][VEC];
    float sum[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int c = (i * blockDim.x + threadIdx.x) * VEC;
        if (live && c < a.cols) {
            load_vec<DT, VEC>(a.x, row * a.cols + c, x[i]);
#pragma unroll
            for (int j = 0; j < VEC; ++j) sum[0] += x[i][j];
        }
    }
    row_sum<1>(sum, s_sum);
    const float mean = sum[0] / static_cast<float>(a.cols);
    sum[0] = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int c = (i * blockDim.x + threadIdx.x) * VEC;
        if (live && c < a.cols) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                x[i][j] -= mean;
                sum[0] = fmaf(x[i][j], x[i][j], sum[0]);
            }
        }
    }
    row_sum<1>(sum, s_sum);
    const float rstd = 1.0f / sqrtf(sum[0] / static_cast<float>(a.cols) + a.eps);
    if (!live) return;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int c = (i * blockDim.x + threadIdx.x) * VEC;
        if (c >= a.cols) continue;
        float w[VEC], b[VEC];
        if (a.weight) load_vec<DT, VEC>(a.weight, c, w);
        if (a.bias) load_vec<DT, VEC>(a.bias, c, b);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            float y = x[i][j] * rstd;
            if (a.weight) y *= w[j];
            if (a.bias) y += b[j];
            x[i][j] = y;
        }
        store_vec<DT, VEC>(a.out, row * a.cols + c, x[i]);
    }
    if (threadIdx.x == 0) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
    }
}

// Rows wider than the registers of a block: the row is read once per pass.
template <int DT>
__global__ void __launch_bounds__(1024) norm_forward_wide_kernel(const NormArgs a) {
    __shared__ float s_sum[32];
    const int64_t base = static_cast<int64_t>(blockIdx.x) * a.cols;
    float f[1], sum[1] = {0.0f};
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
        load_vec<DT, 1>(a.x, base + c, f);
        sum[0] += f[0];
    }
    row_sum<1>(sum, s_sum);
    const float mean = sum[0] / static_cast<float>(a.cols);
    sum[0] = 0.0f;
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
        load_vec<DT, 1>(a.x, base + c, f);
        sum[0] = fmaf(f[0] - mean, f[0] - mean, sum[0]);
    }
    row_sum<1>(sum, s_sum);
    const float rstd = 1.0f / sqrtf(sum[0] / static_cast<float>(a.cols) + a.eps);
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
        float w[1], b[1];
        load_vec<DT, 1>(a.x, base + c, f);
        f[0] = (f[0] - mean) * rstd;
        if (a.weight) {
            load_vec<DT, 1>(a.weight, c, w);
            f[0] *= w[0];
        }
        if (a.bias) {
            load_vec<DT, 1>(a.bias, c, b);
            f[0] += b[0];
        }
        store_vec<DT, 1>(a.out, base + c, f);
    }
    if (threadIdx.x == 0) {
        a.mean[blockIdx.x] = mean;
        a.rstd[blockIdx.x] = rstd;
    }
}

// A block walks over the rows of its group (row = group, group + groups, ...) and keeps the two column sums of its
// columns in registers; they go to the group's partial sums at the end.
template <int DT, int VEC, int VPT>
__global__ void __launch_bounds__(512) norm_backward_kernel(const NormArgs a) {
    __shared__ float s_sum[2 * 32];
    float w[VPT][VEC], dw[VPT][VEC], db[VPT][VEC];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int c = (i * blockDim.x + threadIdx.x) * VEC;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            w[i][j] = 1.0f;
            dw[i][j] = db[i][j] = 0.0f;
        }
        if (a.weight && c < a.cols) load_vec<DT, VEC>(a.weight, c, w[i]);
    }
    const float inv = 1.0f / static_cast<float>(a.cols);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const float mean = a.mean[row], rstd = a.rstd[row];
        float xhat[VPT][VEC], dy[VPT][VEC];
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = (i * blockDim.x + threadIdx.x) * VEC;
            if (c >= a.cols) continue;
            load_vec<DT, VEC>(a.x, row * a.cols + c, xhat[i]);
            load_vec<DT, VEC>(a.dy, row * a.cols + c, dy[i]);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                xhat[i][j] = (xhat[i][j] - mean) * rstd;
                dw[i][j] = fmaf(dy[i][j], xhat[i][j], dw[i][j]);
                db[i][j] += dy[i][j];
                dy[i][j] *= w[i][j];
                sum[0] += dy[i][j];
                sum[1] = fmaf(dy[i][j], xhat[i][j], sum[1]);
            }
        }
        row_sum<2>(sum, s_sum);
        const float m0 = sum[0] * inv, m1 = sum[1] * inv;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = (i * blockDim.x + threadIdx.x) * VEC;
            if (c >= a.cols) continue;
#pragma unroll
            for (int j = 0; j < VEC; ++j) dy[i][j] = rstd * (dy[i][j] - m0 - xhat[i][j] * m1);
            store_vec<DT, VEC>(a.out, row * a.cols + c, dy[i]);
        }
    }
    if (!a.partial) return;
    float* part = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.cols;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int c = (i * blockDim.x + threadIdx.x) * VEC;
        if (c >= a.cols) continue;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            part[c + j] = dw[i][j];
            part[a.cols + c + j] = db[i][j];
        }
    }
}

// Wide rows: dx row by row, and the column sums in a pass of their own.
template <int DT>
__global__ void __launch_bounds__(1024) norm_backward_wide_kernel(const NormArgs a) {
    __shared__ float s_sum[2 * 32];
    const int64_t row = blockIdx.x, base = row * a.cols;
    const float mean = a.mean[row], rstd = a.rstd[row], inv = 1.0f / static_cast<float>(a.cols);
    float x[1], dy[1], w[1] = {1.0f}, sum[2] = {0.0f, 0.0f};
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
        load_vec<DT, 1>(a.x, base + c, x);
        load_vec<DT, 1>(a.dy, base + c, dy);
        if (a.weight) load_vec<DT, 1>(a.weight, c, w);
        sum[0] += dy[0] * w[0];
        sum[1] = fmaf(dy[0] * w[0], (x[0] - mean) * rstd, sum[1]);
    }
    row_sum<2>(sum, s_sum);
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
        load_vec<DT, 1>(a.x, base + c, x);
        load_vec<DT, 1>(a.dy, base + c, dy);
        if (a.weight) load_vec<DT, 1>(a.weight, c, w);
        x[0] = rstd * (dy[0] * w[0] - sum[0] * inv - (x[0] - mean) * rstd * (sum[1] * inv));
        store_vec<DT, 1>(a.out, base + c, x);
    }
}
template <int DT>
__global__ void __launch_bounds__(256) norm_columns_wide_kernel(const NormArgs a) {
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= a.cols) return;
    float dw = 0.0f, db = 0.0f, x[1], dy[1];
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        load_vec<DT, 1>(a.x, row * a.cols + c, x);
        load_vec<DT, 1>(a.dy, row * a.cols + c, dy);
        dw = fmaf(dy[0], (x[0] - a.mean[row]) * a.rstd[row], dw);
        db += dy[0];
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

template <int DT, int VEC, int VPT>
int launch_forward(const NormArgs& a, cudaStream_t s) {
    const int threads = round32((a.cols + VEC * VPT - 1) / (VEC * VPT));
    const int per_block = threads >= 256 ? 1 : min(kMaxRowsPerBlock, 256 / threads);
    const int64_t grid = (a.rows + per_block - 1) / per_block;
    if (grid > 0x7FFFFFFF) return ELX_ERR_CAPACITY;
    norm_forward_kernel<DT, VEC, VPT><<<static_cast<unsigned>(grid), dim3(threads, per_block), 0, s>>>(a);
    return record_cuda(cudaGetLastError());
}

template <int DT>
int forward_dt(const NormArgs& a, bool wide_ok, cudaStream_t s) {
    constexpr int V = Wide<DT>::kVec;
    if (wide_ok) {
        const int vecs = a.cols / V;
        if (vecs <= 512) return launch_forward<DT, V, 1>(a, s);
        if (vecs <= 1024) return launch_forward<DT, V, 2>(a, s);
        if (vecs <= 4096) return launch_forward<DT, V, 4>(a, s);
    } else {
        if (a.cols <= 512) return launch_forward<DT, 1, 2>(a, s);
        if (a.cols <= 4096) return launch_forward<DT, 1, 8>(a, s);
        if (a.cols <= 16384) return launch_forward<DT, 1, 16>(a, s);
    }
    if (a.rows > 0x7FFFFFFF) return ELX_ERR_CAPACITY;
    norm_forward_wide_kernel<DT><<<static_cast<unsigned>(a.rows), 1024, 0, s>>>(a);
    return record_cuda(cudaGetLastError());
}

int backward_groups(int64_t rows) { return static_cast<int>(rows < 592 ? rows : 592); }

template <int DT, int VEC, int VPT>
int launch_backward(const NormArgs& a, cudaStream_t s) {
    const int threads = round32((a.cols + VEC * VPT - 1) / (VEC * VPT));
    norm_backward_kernel<DT, VEC, VPT><<<a.groups, threads, 0, s>>>(a);
    return record_cuda(cudaGetLastError());
}

template <int DT>
int backward_dt(const NormArgs& a, bool wide_ok, void* dweight, void* dbias, cudaStream_t s) {
    constexpr int V = Wide<DT>::kVec;
    int rc = 1;
    if (wide_ok) {
        const int vecs = a.cols / V;
        if (vecs <= 128) rc = launch_backward<DT, V, 1>(a, s);
        else if (vecs <= 1024) rc = launch_backward<DT, V, 2>(a, s);
    } else {
        if (a.cols <= 512) rc = launch_backward<DT, 1, 2>(a, s);
        else if (a.cols <= 4096) rc = launch_backward<DT, 1, 8>(a, s);
    }
    if (rc == 1) {
        if (a.rows > 0x7FFFFFFF) return ELX_ERR_CAPACITY;
        norm_backward_wide_kernel<DT><<<static_cast<unsigned>(a.rows), 1024, 0, s>>>(a);
        rc = record_cuda(cudaGetLastError());
        if (rc == ELX_OK && a.partial) {
            norm_columns_wide_kernel<DT><<<dim3((a.cols + 255) / 256, a.groups), 256, 0, s>>>(a);
            rc = record_cuda(cudaGetLastError());
        }
    }
    if (rc != ELX_OK || !a.partial) return rc;
    norm_columns_kernel<DT><<<(a.cols + 31) / 32, dim3(32, 32), 0, s>>>(a.partial, a.groups, a.cols, dweight, dbias);
    return record_cuda(cudaGetLastError());
}

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
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case ELX_F16: return forward_dt<ELX_F16>(a, wide_ok, s);
        case ELX_BF16: return forward_dt<ELX_BF16>(a, wide_ok, s);
    }
    return forward_dt<ELX_F32>(a, wide_ok, s);
}

int64_t elx_layer_norm_backward_workspace(int64_t rows, int64_t cols) {
    if (rows < 0 || cols <= 0) return ELX_ERR_SIZE;
    return static_cast<int64_t>(backward_groups(rows)) * 2 * cols * 4;
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
    a.groups = backward_groups(rows);
    const bool wide_ok = cols * size % 16 == 0 && aligned(x, 16) && aligned(dy, 16) && aligned(dx, 16) && aligned(weight, 16);
    switch (dtype) {
        case ELX_F16: return backward_dt<ELX_F16>(a, wide_ok, dweight, dbias, s);
        case ELX_BF16: return backward_dt<ELX_BF16>(a, wide_ok, dweight, dbias, s);
    }
    return backward_dt<ELX_F32>(a, wide_ok, dweight, dbias, s);
}

}  // extern "C"
