// Part of the elixir_b200 CUDA library (C ABI: include/elixir_b200.h): embedding lookup with a scale, and its gradient.
//
//   out[i] = scale * weight[token i]
//   dweight[v] = scale * sum over i ascending with token i == v, v not the padding token, of dout[i]
//
// The gradient adds in fp32, in an order that the inputs alone fix: the tokens are sorted (stably, by radix), the
// sorted positions are cut into pieces of 32, a piece sums its runs of equal tokens, and a run that spans pieces is
// put together from their partial sums in order.  No floating-point atomics.
//
// A token outside [0, vocab) looks up a row of NaN (the loss, the gradients and the overflow probe then see it) and
// adds to no row of the gradient.
#include "elx_common.cuh"

using namespace elx;

namespace {

constexpr int kEmbedThreads = 256;

template <typename I>
__device__ __forceinline__ int64_t token_at(const void* tokens, int64_t i) {
    return static_cast<int64_t>(static_cast<const I*>(tokens)[i]);
}

// VEC elements scaled in fp32 and rounded once; a scale of 1 moves the bits.
template <int DT, int VEC, typename I>
__global__ void __launch_bounds__(kEmbedThreads) embed_forward_kernel(const void* tokens, int64_t n, const void* weight,
                                                                      int64_t vocab, int64_t width, float scale, void* out) {
    using T = typename Lp<DT>::T;
    const int64_t per_row = width / VEC, total = n * per_row;
    for (int64_t at = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; at < total;
         at += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int64_t row = at / per_row, c = (at - row * per_row) * VEC;
        const int64_t v = token_at<I>(tokens, row);
        const bool good = v >= 0 && v < vocab;
        if constexpr (VEC == 1) {
            const float f = good ? Lp<DT>::to_float(static_cast<const T*>(weight)[v * width + c]) * scale : __int_as_float(0x7FC00000);
            static_cast<T*>(out)[row * width + c] = Lp<DT>::from_float(f);
        } else {
            uint4 r;
            uint32_t w[4];
            if (good) {
                r = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(weight) + v * width + c));
                w[0] = r.x; w[1] = r.y; w[2] = r.z; w[3] = r.w;
                if (scale != 1.0f) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if constexpr (DT == ELX_F32) {
                            w[j] = __float_as_uint(__uint_as_float(w[j]) * scale);
                        } else {
                            const float2 f = Lp<DT>::unpack2(w[j]);
                            w[j] = Lp<DT>::pack2(f.x * scale, f.y * scale);
                        }
                    }
                }
            } else {
                const uint32_t nan = DT == ELX_F32 ? 0x7FC00000u : DT == ELX_F16 ? 0x7E007E00u : 0x7FC07FC0u;
                w[0] = w[1] = w[2] = w[3] = nan;
            }
            *reinterpret_cast<uint4*>(static_cast<T*>(out) + row * width + c) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

// ------------------------------------------------------------------------------------------------
// stable radix sort of (token, position), 8 bits per pass
// ------------------------------------------------------------------------------------------------

constexpr int kSortThreads = 256, kSortItems = 8, kSortTile = kSortThreads * kSortItems, kDigits = 256;

// Tokens that add to no row get the key `vocab` and sort behind the others.
template <typename I>
__global__ void __launch_bounds__(kSortThreads) embed_keys_kernel(const void* tokens, int64_t n, int64_t vocab, int64_t padding,
                                                                  uint32_t* keys, uint32_t* order) {
    const int64_t i = blockIdx.x * static_cast<int64_t>(kSortThreads) + threadIdx.x;
    if (i >= n) return;
    const int64_t v = token_at<I>(tokens, i);
    keys[i] = static_cast<uint32_t>(v >= 0 && v < vocab && v != padding ? v : vocab);
    order[i] = static_cast<uint32_t>(i);
}

__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(const uint32_t* __restrict__ keys, int64_t n, int shift,
                                                                  uint32_t* counts) {
    __shared__ uint32_t s_count[kDigits];
    s_count[threadIdx.x] = 0;
    __syncthreads();
    const int64_t base = blockIdx.x * static_cast<int64_t>(kSortTile);
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        const int64_t i = base + k * kSortThreads + threadIdx.x;
        if (i < n) atomicAdd(&s_count[(keys[i] >> shift) & 0xFFu], 1u);
    }
    __syncthreads();
    counts[static_cast<int64_t>(threadIdx.x) * gridDim.x + blockIdx.x] = s_count[threadIdx.x];
}

// Exclusive prefix sum of `n` counters, in place, by one block.
__global__ void __launch_bounds__(1024) sort_scan_kernel(uint32_t* counts, int64_t n) {
    __shared__ uint32_t s_warp[32];
    __shared__ uint32_t s_carry;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) s_carry = 0;
    __syncthreads();
    for (int64_t base = 0; base < n; base += 1024) {
        const int64_t i = base + threadIdx.x;
        const uint32_t mine = i < n ? counts[i] : 0u;
        uint32_t inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t up = __shfl_up_sync(0xFFFFFFFFu, inc, o);
            if (lane >= o) inc += up;
        }
        if (lane == 31) s_warp[warp] = inc;
        __syncthreads();
        if (warp == 0) {
            uint32_t t = s_warp[lane];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t up = __shfl_up_sync(0xFFFFFFFFu, t, o);
                if (lane >= o) t += up;
            }
            s_warp[lane] = t;
        }
        __syncthreads();
        const uint32_t before = s_carry + (warp ? s_warp[warp - 1] : 0u) + inc - mine;
        if (i < n) counts[i] = before;
        __syncthreads();
        if (threadIdx.x == 0) s_carry += s_warp[31];
        __syncthreads();
    }
}

// A warp owns 256 consecutive items of the tile, 32 at a time, so an item's place among the equal digits of its tile
// is (those of earlier warps) + (those of earlier rounds) + (those of lower lanes).
__global__ void __launch_bounds__(kSortThreads) sort_scatter_kernel(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ order,
                                                                    int64_t n, int shift, const uint32_t* __restrict__ starts,
                                                                    uint32_t* keys_out, uint32_t* order_out) {
    constexpr int kWarps = kSortThreads / 32;
    __shared__ uint32_t s_place[kWarps][kDigits];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int i = threadIdx.x; i < kWarps * kDigits; i += kSortThreads) (&s_place[0][0])[i] = 0;
    __syncthreads();
    const int64_t base = blockIdx.x * static_cast<int64_t>(kSortTile) + warp * (kSortItems * 32);
    uint32_t key[kSortItems], rank[kSortItems];
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        const int64_t i = base + k * 32 + lane;
        const bool live = i < n;
        key[k] = live ? keys[i] : 0u;
        const uint32_t digit = live ? (key[k] >> shift) & 0xFFu : 0xFFFFFFFFu;
        const uint32_t same = __match_any_sync(0xFFFFFFFFu, digit);
        const uint32_t seen = live ? s_place[warp][digit] : 0u;
        rank[k] = seen + __popc(same & ((1u << lane) - 1u));
        __syncwarp();
        if (live && lane == __ffs(same) - 1) s_place[warp][digit] = seen + __popc(same);
        __syncwarp();
    }
    __syncthreads();
    {
        uint32_t t = starts[static_cast<int64_t>(threadIdx.x) * gridDim.x + blockIdx.x];
        for (int w = 0; w < kWarps; ++w) {
            const uint32_t here = s_place[w][threadIdx.x];
            s_place[w][threadIdx.x] = t;
            t += here;
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        const int64_t i = base + k * 32 + lane;
        if (i >= n) continue;
        const uint32_t to = s_place[warp][(key[k] >> shift) & 0xFFu] + rank[k];
        keys_out[to] = key[k];
        order_out[to] = order[i];
    }
}

// ------------------------------------------------------------------------------------------------
// sums
// ------------------------------------------------------------------------------------------------

constexpr int kPiece = 32;   // sorted positions per piece

template <int DT, int VEC>
__device__ __forceinline__ void add_vec(const void* base, int64_t i, float (&acc)[VEC]) {
    using T = typename Lp<DT>::T;
    if constexpr (VEC == 1) {
        acc[0] += Lp<DT>::to_float(static_cast<const T*>(base)[i]);
    } else {
        const uint4 r = *reinterpret_cast<const uint4*>(static_cast<const T*>(base) + i);
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (DT == ELX_F32) {
                acc[j] += __uint_as_float(w[j]);
            } else {
                const float2 f = Lp<DT>::unpack2(w[j]);
                acc[2 * j] += f.x;
                acc[2 * j + 1] += f.y;
            }
        }
    }
}
template <int DT, int VEC>
__device__ __forceinline__ void store_scaled(void* base, int64_t i, const float (&acc)[VEC], float scale) {
    using T = typename Lp<DT>::T;
    if constexpr (VEC == 1) {
        static_cast<T*>(base)[i] = Lp<DT>::from_float(acc[0] * scale);
    } else if constexpr (DT == ELX_F32) {
        *reinterpret_cast<float4*>(static_cast<T*>(base) + i) =
            make_float4(acc[0] * scale, acc[1] * scale, acc[2] * scale, acc[3] * scale);
    } else {
        *reinterpret_cast<uint4*>(static_cast<T*>(base) + i) =
            make_uint4(Lp<DT>::pack2(acc[0] * scale, acc[1] * scale), Lp<DT>::pack2(acc[2] * scale, acc[3] * scale),
                       Lp<DT>::pack2(acc[4] * scale, acc[5] * scale), Lp<DT>::pack2(acc[6] * scale, acc[7] * scale));
    }
}

// partial: two rows of fp32 sums per piece -- slot 0 for a run that began in an earlier piece, slot 1 for one that
// begins here and goes on in the next.
template <int DT, int VEC>
__global__ void __launch_bounds__(kEmbedThreads) embed_sum_kernel(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ order,
                                                                  int64_t n, const void* __restrict__ dout, int64_t vocab,
                                                                  int64_t width, float scale, void* dweight, float* partial) {
    __shared__ uint32_t s_key[kPiece + 2];    // with the neighbours on both sides
    __shared__ uint32_t s_pos[kPiece];
    const int64_t first = blockIdx.x * static_cast<int64_t>(kPiece);
    const uint32_t none = 0xFFFFFFFFu;        // larger than any key
    if (threadIdx.x < kPiece + 2) {
        const int64_t i = first + threadIdx.x - 1;
        s_key[threadIdx.x] = i >= 0 && i < n ? keys[i] : none;
    }
    if (threadIdx.x < kPiece) s_pos[threadIdx.x] = first + threadIdx.x < n ? order[first + threadIdx.x] : 0u;
    __syncthreads();
    const int live = static_cast<int>(min(static_cast<int64_t>(kPiece), n - first));
    for (int64_t c = (blockIdx.y * static_cast<int64_t>(blockDim.x) + threadIdx.x) * VEC; c < width;
         c += static_cast<int64_t>(gridDim.y) * blockDim.x * VEC) {
        for (int p = 0; p < live;) {
            const uint32_t key = s_key[p + 1];
            if (key >= vocab) break;          // padding and tokens out of range: the last keys
            const bool begins = s_key[p] != key;
            float acc[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
            do {
                add_vec<DT, VEC>(dout, static_cast<int64_t>(s_pos[p]) * width + c, acc);
                ++p;
            } while (p < live && s_key[p + 1] == key);
            const bool ends = p < live || s_key[live + 1] != key;
            if (begins && ends) {
                store_scaled<DT, VEC>(dweight, static_cast<int64_t>(key) * width + c, acc, scale);
            } else {
                float* const to = partial + (blockIdx.x * 2 + (begins ? 1 : 0)) * width + c;
#pragma unroll
                for (int j = 0; j < VEC; ++j) to[j] = acc[j];
            }
        }
    }
}

// The runs that span pieces: the piece in which a run begins adds up the partial sums of the pieces that it reaches.
template <int DT, int VEC>
__global__ void __launch_bounds__(kEmbedThreads) embed_join_kernel(const uint32_t* __restrict__ keys, int64_t n, int64_t vocab,
                                                                   int64_t width, float scale, void* dweight,
                                                                   const float* __restrict__ partial) {
    const int64_t piece = blockIdx.x, last = piece * kPiece + kPiece - 1;
    if (last + 1 >= n) return;                       // the last piece: nothing goes on
    const uint32_t key = keys[last];
    if (key >= vocab || keys[last + 1] != key) return;
    // begins here?  (the run may fill the whole piece and come from an earlier one)
    if (piece > 0 && keys[piece * kPiece] == key && keys[piece * kPiece - 1] == key) return;
    for (int64_t c = (blockIdx.y * static_cast<int64_t>(blockDim.x) + threadIdx.x) * VEC; c < width;
         c += static_cast<int64_t>(gridDim.y) * blockDim.x * VEC) {
        float acc[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] = partial[(piece * 2 + 1) * width + c + j];
        for (int64_t q = piece + 1; q * kPiece < n && keys[q * kPiece] == key; ++q)
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[j] += partial[q * 2 * width + c + j];
        store_scaled<DT, VEC>(dweight, static_cast<int64_t>(key) * width + c, acc, scale);
    }
}

int64_t align16(int64_t n) { return (n + 15) / 16 * 16; }

struct EmbedSpace {
    int64_t keys, counts, partial, total;   // bytes: one key or position array, the counters, the partial sums
};
EmbedSpace embed_space(int64_t n, int64_t width) {
    EmbedSpace s;
    s.keys = align16(n * 4);
    s.counts = align16((n + kSortTile - 1) / kSortTile * kDigits * 4);
    s.partial = align16((n + kPiece - 1) / kPiece * 2 * width * 4);
    s.total = 4 * s.keys + s.counts + s.partial;
    return s;
}

template <int DT, int VEC>
int launch_sums(const uint32_t* keys, const uint32_t* order, int64_t n, const void* dout, int64_t vocab, int64_t width, float scale,
                void* dweight, float* partial, cudaStream_t s) {
    const int64_t pieces = (n + kPiece - 1) / kPiece;
    const int64_t slabs = (width + VEC * kEmbedThreads - 1) / (VEC * kEmbedThreads);
    const dim3 grid(static_cast<unsigned>(pieces), static_cast<unsigned>(slabs < 64 ? slabs : 64));
    embed_sum_kernel<DT, VEC><<<grid, kEmbedThreads, 0, s>>>(keys, order, n, dout, vocab, width, scale, dweight, partial);
    embed_join_kernel<DT, VEC><<<grid, kEmbedThreads, 0, s>>>(keys, n, vocab, width, scale, dweight, partial);
    return record_cuda(cudaGetLastError());
}

template <int DT>
int forward_dt(const void* tokens, int index_bytes, int64_t n, const void* weight, int64_t vocab, int64_t width, float scale,
               void* out, cudaStream_t s) {
    constexpr int V = DT == ELX_F32 ? 4 : 8;
    const bool wide = width % V == 0 && aligned(weight, 16) && aligned(out, 16);
    const int64_t items = n * (wide ? width / V : width);
    const int grid = grid_for((items + kEmbedThreads - 1) / kEmbedThreads, 16);
    if (grid < 0) return grid;
    if (wide) {
        if (index_bytes == 8) embed_forward_kernel<DT, V, int64_t><<<grid, kEmbedThreads, 0, s>>>(tokens, n, weight, vocab, width, scale, out);
        else embed_forward_kernel<DT, V, int32_t><<<grid, kEmbedThreads, 0, s>>>(tokens, n, weight, vocab, width, scale, out);
    } else {
        if (index_bytes == 8) embed_forward_kernel<DT, 1, int64_t><<<grid, kEmbedThreads, 0, s>>>(tokens, n, weight, vocab, width, scale, out);
        else embed_forward_kernel<DT, 1, int32_t><<<grid, kEmbedThreads, 0, s>>>(tokens, n, weight, vocab, width, scale, out);
    }
    return record_cuda(cudaGetLastError());
}

int check_embedding(const void* tokens, int index_bytes, int64_t n, int dtype, int64_t vocab, int64_t width, const void* a,
                    const void* b) {
    if (n < 0 || vocab <= 0 || width <= 0) return ELX_ERR_SIZE;
    if (n > 0 && !tokens) return ELX_ERR_NULL;
    if (!dtype_ok(dtype) || (index_bytes != 4 && index_bytes != 8)) return ELX_ERR_DTYPE;
    if (n > 0x7FFFFFFFll || vocab > 0x7FFFFFFFll || width > 0x7FFFFFFFll) return ELX_ERR_CAPACITY;
    const int size = dtype_bytes(dtype);
    if (!aligned(tokens, index_bytes) || !aligned(a, size) || !aligned(b, size)) return ELX_ERR_ALIGN;
    return ELX_OK;
}

}  // namespace

extern "C" {

int elx_embedding_forward(const void* tokens, int index_bytes, int64_t n, const void* weight, int dtype, int64_t vocab,
                          int64_t width, float scale, void* out, void* stream) {
    if (!weight || (n > 0 && !out)) return ELX_ERR_NULL;
    const int rc = check_embedding(tokens, index_bytes, n, dtype, vocab, width, weight, out);
    if (rc != ELX_OK || n == 0) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case ELX_F16: return forward_dt<ELX_F16>(tokens, index_bytes, n, weight, vocab, width, scale, out, s);
        case ELX_BF16: return forward_dt<ELX_BF16>(tokens, index_bytes, n, weight, vocab, width, scale, out, s);
    }
    return forward_dt<ELX_F32>(tokens, index_bytes, n, weight, vocab, width, scale, out, s);
}

int64_t elx_embedding_backward_workspace(int64_t n, int64_t width) {
    if (n < 0 || width <= 0) return ELX_ERR_SIZE;
    return embed_space(n, width).total;
}

int elx_embedding_backward(const void* tokens, int index_bytes, int64_t n, const void* dout, int dtype, int64_t vocab,
                           int64_t width, float scale, int64_t padding_idx, void* dweight, void* workspace,
                           int64_t workspace_bytes, void* stream) {
    if (!dweight || (n > 0 && !dout)) return ELX_ERR_NULL;
    const int rc = check_embedding(tokens, index_bytes, n, dtype, vocab, width, dout, dweight);
    if (rc != ELX_OK) return rc;
    if (padding_idx < -1 || padding_idx >= vocab) return ELX_ERR_ARG;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const EmbedSpace space = embed_space(n, width);
    if (n > 0) {
        if (!workspace) return ELX_ERR_NULL;
        if (!aligned(workspace, 16)) return ELX_ERR_ALIGN;
        if (workspace_bytes < space.total) return ELX_ERR_CAPACITY;
    }
    const int size = dtype_bytes(dtype);
    const cudaError_t zeroed = cudaMemsetAsync(dweight, 0, vocab * width * size, s);
    if (zeroed != cudaSuccess) return record_cuda(zeroed);
    if (n == 0) return ELX_OK;
    char* at = static_cast<char*>(workspace);
    uint32_t *keys[2], *order[2];
    for (int k = 0; k < 2; ++k, at += 2 * space.keys) {
        keys[k] = reinterpret_cast<uint32_t*>(at);
        order[k] = reinterpret_cast<uint32_t*>(at + space.keys);
    }
    uint32_t* const counts = reinterpret_cast<uint32_t*>(at);
    float* const partial = reinterpret_cast<float*>(at + space.counts);
    const unsigned fill = static_cast<unsigned>((n + kSortThreads - 1) / kSortThreads);
    if (index_bytes == 8) embed_keys_kernel<int64_t><<<fill, kSortThreads, 0, s>>>(tokens, n, vocab, padding_idx, keys[0], order[0]);
    else embed_keys_kernel<int32_t><<<fill, kSortThreads, 0, s>>>(tokens, n, vocab, padding_idx, keys[0], order[0]);
    const unsigned tiles = static_cast<unsigned>((n + kSortTile - 1) / kSortTile);
    int from = 0;
    for (int shift = 0; shift < 32 && (vocab >> shift) != 0; shift += 8, from ^= 1) {
        sort_count_kernel<<<tiles, kSortThreads, 0, s>>>(keys[from], n, shift, counts);
        sort_scan_kernel<<<1, 1024, 0, s>>>(counts, static_cast<int64_t>(tiles) * kDigits);
        sort_scatter_kernel<<<tiles, kSortThreads, 0, s>>>(keys[from], order[from], n, shift, counts, keys[from ^ 1], order[from ^ 1]);
    }
    const uint32_t *k = keys[from], *o = order[from];
    const bool wide16 = width % 8 == 0 && aligned(dout, 16) && aligned(dweight, 16);
    const bool wide32 = width % 4 == 0 && aligned(dout, 16) && aligned(dweight, 16);
    switch (dtype) {
        case ELX_F16:
            return wide16 ? launch_sums<ELX_F16, 8>(k, o, n, dout, vocab, width, scale, dweight, partial, s)
                          : launch_sums<ELX_F16, 1>(k, o, n, dout, vocab, width, scale, dweight, partial, s);
        case ELX_BF16:
            return wide16 ? launch_sums<ELX_BF16, 8>(k, o, n, dout, vocab, width, scale, dweight, partial, s)
                          : launch_sums<ELX_BF16, 1>(k, o, n, dout, vocab, width, scale, dweight, partial, s);
    }
    return wide32 ? launch_sums<ELX_F32, 4>(k, o, n, dout, vocab, width, scale, dweight, partial, s)
                  : launch_sums<ELX_F32, 1>(k, o, n, dout, vocab, width, scale, dweight, partial, s);
}

}  // extern "C"
