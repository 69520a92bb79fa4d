// Part of the elixir_b200 CUDA library (C ABI: include/elixir_b200.h): embedding lookup with a scale, and its gradient.
//
//   out[i] = scale * weight[token i]
//   dweight[v] = scale * sum over i ascending with token i == v, v not the padding token, of dout[i]
//
// The gradient adds in fp32, in an order that the inputs alone fix: the tokens are sorted (stably, by radix), the
// sorted positions are cut into pieces of 32, a piece sums its runs of equal tokens, and a run that spans pieces is
// put together from their partial sums in order.  No floating-point atomics.  Three launches: the sort by one cluster of
// eight blocks while all other blocks write the zeros of the table's rows, the sums, the joining of long runs.
//
// A token outside [0, vocab) looks up a row of NaN (the loss, the gradients and the overflow probe then see it) and
// adds to no row of the gradient.
#include <cooperative_groups.h>

#include "elx_common.cuh"

using namespace elx;

namespace {

constexpr int kEmbedThreads = 256;
constexpr int kMostRows = 32;   // rows (or pieces of the sorted tokens) that a block works on side by side

template <typename I>
__device__ __forceinline__ int64_t token_at(const void* tokens, int64_t i) {
    return static_cast<int64_t>(static_cast<const I*>(tokens)[i]);
}

// VEC elements of a row as they are held in memory: 16 bytes, 4 bytes (two 16-bit elements), or one element.
template <int DT, int VEC>
struct Bits {
    static constexpr int kBytes = VEC * Lp<DT>::kBytes, kWords = kBytes >= 4 ? kBytes / 4 : 1;
    static_assert(kBytes == 16 || kBytes == 4 || kBytes == 2, "16 bytes, a word or a 16-bit element");
    uint32_t w[kWords];
    __device__ __forceinline__ void load(const void* base, int64_t element) {
        const char* const p = static_cast<const char*>(base) + element * Lp<DT>::kBytes;
        if constexpr (kBytes == 16) {
            const uint4 r = *reinterpret_cast<const uint4*>(p);
            w[0] = r.x; w[1] = r.y; w[2] = r.z; w[3] = r.w;
        } else if constexpr (kBytes == 4) {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        } else {
            w[0] = *reinterpret_cast<const uint16_t*>(p);
        }
    }
    __device__ __forceinline__ void store(void* base, int64_t element) const {
        char* const p = static_cast<char*>(base) + element * Lp<DT>::kBytes;
        if constexpr (kBytes == 16) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        else if constexpr (kBytes == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
        else *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(w[0]);
    }
    __device__ __forceinline__ void get(float (&f)[VEC]) const {
        if constexpr (DT == ELX_F32) {
#pragma unroll
            for (int j = 0; j < kWords; ++j) f[j] = __uint_as_float(w[j]);
        } else if constexpr (VEC == 1) {
            f[0] = Lp<DT>::unpack2(w[0]).x;
        } else {
#pragma unroll
            for (int j = 0; j < kWords; ++j) {
                const float2 p = Lp<DT>::unpack2(w[j]);
                f[2 * j] = p.x;
                f[2 * j + 1] = p.y;
            }
        }
    }
    __device__ __forceinline__ void put(const float (&f)[VEC]) {
        if constexpr (DT == ELX_F32) {
#pragma unroll
            for (int j = 0; j < kWords; ++j) w[j] = __float_as_uint(f[j]);
        } else if constexpr (VEC == 1) {
            w[0] = Lp<DT>::pack2(f[0], 0.0f);
        } else {
#pragma unroll
            for (int j = 0; j < kWords; ++j) w[j] = Lp<DT>::pack2(f[2 * j], f[2 * j + 1]);
        }
    }
    __device__ __forceinline__ void nan() {
#pragma unroll
        for (int j = 0; j < kWords; ++j) w[j] = DT == ELX_F32 ? 0x7FC00000u : DT == ELX_F16 ? 0x7E007E00u : 0x7FC07FC0u;
    }
};

// A row per blockDim.x threads, blockDim.y rows per block; four accesses of a thread on their way at a time.  Scaled in fp32
// and rounded once; a scale of 1 moves the bits.
template <int DT, int VEC, typename I>
__global__ void __launch_bounds__(kEmbedThreads) embed_forward_kernel(const void* tokens, int64_t n, const void* weight,
                                                                      int64_t vocab, int width, float scale, void* out) {
    const int pieces = width / VEC;
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y; row < n;
         row += static_cast<int64_t>(gridDim.x) * blockDim.y) {
        const int64_t v = token_at<I>(tokens, row);
        const bool good = v >= 0 && v < vocab;
        const int64_t from = good ? v * width : 0, to = row * width;
        for (int p0 = threadIdx.x; p0 < pieces; p0 += 4 * blockDim.x) {
            Bits<DT, VEC> b[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int p = p0 + k * blockDim.x;
                if (p < pieces) b[k].load(weight, from + static_cast<int64_t>(p) * VEC);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int p = p0 + k * blockDim.x;
                if (p >= pieces) break;
                if (!good) {
                    b[k].nan();
                } else if (scale != 1.0f) {
                    float f[VEC];
                    b[k].get(f);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) f[j] *= scale;
                    b[k].put(f);
                }
                b[k].store(out, to + static_cast<int64_t>(p) * VEC);
            }
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

// Exclusive prefix sum of `n` counters (a multiple of eight), in place, by one block; eight counters per thread and round, the
// next round's on their way meanwhile.
__global__ void __launch_bounds__(1024) sort_scan_kernel(uint32_t* counts, int64_t n) {
    __shared__ uint32_t s_warp[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    uint4* const at4 = reinterpret_cast<uint4*>(counts) + threadIdx.x * 2;
    const int64_t n4 = n / 4 - threadIdx.x * 2;
    uint4 a = n4 > 0 ? at4[0] : zero, b = n4 > 0 ? at4[1] : zero;
    uint32_t carry = 0;
    for (int64_t base = 0; base < n / 4; base += 2 * 1024) {
        uint32_t c[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}, mine = 0;
        if (base + 2 * 1024 < n4) a = at4[base + 2 * 1024], b = at4[base + 2 * 1024 + 1];
        else a = b = zero;
#pragma unroll
        for (int k = 0; k < 8; ++k) mine += c[k];
        uint32_t inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t up = __shfl_up_sync(0xFFFFFFFFu, inc, o);
            if (lane >= o) inc += up;
        }
        __syncthreads();   // the round before has been read
        if (lane == 31) s_warp[warp] = inc;
        __syncthreads();
        uint32_t t = s_warp[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t up = __shfl_up_sync(0xFFFFFFFFu, t, o);
            if (lane >= o) t += up;
        }
        const uint32_t before_warp = __shfl_sync(0xFFFFFFFFu, t, (warp + 31) & 31);
        uint32_t at = carry + (warp ? before_warp : 0u) + inc - mine;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t here = c[k];
            c[k] = at;
            at += here;
        }
        if (base < n4) {
            at4[base] = make_uint4(c[0], c[1], c[2], c[3]);
            at4[base + 1] = make_uint4(c[4], c[5], c[6], c[7]);
        }
        carry += __shfl_sync(0xFFFFFFFFu, t, 31);
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
// the same sort by one cluster of eight blocks, in shared memory, next to the zeros of the gradient
// ------------------------------------------------------------------------------------------------
//
// Each block of the first cluster holds C tokens in shared memory (C a power of two, at most 8192).  Eight bits per pass: digits are counted per warp, the blocks tell each other their totals, and every token goes to its
// place in whichever block holds it.  Two cluster barriers per pass, no launch between them: 8192 tokens in about 10 us
// instead of 25 us for the separate launches -- and none of it shows, because the blocks of all other clusters write the
// zeros of the table's rows meanwhile (161 MB for 50257 x 1600 fp16).

constexpr int kCluster = 8, kClusterThreads = 1024, kClusterWarps = 32, kMostPerBlock = 8192;
constexpr int64_t kMostInCluster = static_cast<int64_t>(kCluster) * kMostPerBlock;

struct SortSpace {
    uint32_t place[kClusterWarps][kDigits];   // per warp and digit: how many, then where the next one goes
    uint32_t totals[kCluster][kDigits];       // every block's totals, in every block
    uint32_t scan[8];
};

template <typename I>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kClusterThreads, 1)
    embed_sort_kernel(const void* tokens, int64_t n, int64_t vocab, int64_t padding, int log_c, int passes, uint32_t* keys_out,
                      uint32_t* order_out, char* zeros, int64_t zero_bytes) {
    extern __shared__ __align__(16) uint32_t s_dyn[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (blockIdx.x >= kCluster) {
        // the zeros: 32 bytes per store, the two ends by the byte
        const int64_t blocks = gridDim.x - kCluster, me = blockIdx.x - kCluster;
        const int64_t head = min(static_cast<int64_t>((32 - (reinterpret_cast<uintptr_t>(zeros) & 31u)) & 31u), zero_bytes);
        const int64_t whole = (zero_bytes - head) / 32, tail = zero_bytes - head - 32 * whole;
        char* const at = zeros + head;
        U8 zero;
#pragma unroll
        for (int j = 0; j < 8; ++j) zero.x[j] = 0;
#pragma unroll 4
        for (int64_t i = me * kClusterThreads + threadIdx.x; i < whole; i += blocks * kClusterThreads) st256(at + 32 * i, zero);
        next_may_start();
        if (me == 0 && threadIdx.x < head) zeros[threadIdx.x] = 0;
        if (me == 0 && threadIdx.x < tail) at[32 * whole + threadIdx.x] = 0;
        return;
    }
    cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    const int c = 1 << log_c, rank = static_cast<int>(cluster.block_rank());
    const int rounds = (c + kClusterThreads - 1) / kClusterThreads;           // items per thread
    const int per_warp = c >= kClusterThreads ? c / kClusterWarps : 32;       // consecutive items of a warp
    SortSpace& sp = *reinterpret_cast<SortSpace*>(s_dyn);
    uint32_t* const keys = s_dyn + sizeof(SortSpace) / 4;                     // [2][c]
    uint32_t* const order = keys + 2 * c;                                     // [2][c]
    const int64_t base = static_cast<int64_t>(rank) << log_c;
    const int mine = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(c), n - base)));   // tokens here
    // tokens that add to no row get the key `vocab` and sort behind the others
    for (int i = threadIdx.x; i < mine; i += kClusterThreads) {
        const int64_t v = token_at<I>(tokens, base + i);
        keys[i] = static_cast<uint32_t>(v >= 0 && v < vocab && v != padding ? v : vocab);
        order[i] = static_cast<uint32_t>(base + i);
    }
    cluster.sync();
    int from = 0;
    for (int pass = 0; pass < passes; ++pass, from ^= 1) {
        const int shift = 8 * pass;
        const uint32_t *const k_in = keys + from * c, *const o_in = order + from * c;
        for (int i = threadIdx.x; i < kClusterWarps * kDigits; i += kClusterThreads) (&sp.place[0][0])[i] = 0;
        __syncthreads();
        // a warp owns consecutive items, 32 at a time: places among equal digits follow the tokens' order
        uint32_t key[kMostPerBlock / kClusterThreads], rank_in[kMostPerBlock / kClusterThreads];
#pragma unroll
        for (int r = 0; r < kMostPerBlock / kClusterThreads; ++r) {
            if (r >= rounds) break;
            const int i = warp * per_warp + r * 32 + lane;
            const bool live = i < mine;
            key[r] = live ? k_in[i] : 0u;
            const uint32_t digit = live ? (key[r] >> shift) & 0xFFu : 0xFFFFFFFFu;
            const uint32_t same = __match_any_sync(0xFFFFFFFFu, digit);
            const uint32_t seen = live ? sp.place[warp][digit] : 0u;
            rank_in[r] = seen + __popc(same & ((1u << lane) - 1u));
            __syncwarp();
            if (live && lane == __ffs(same) - 1) sp.place[warp][digit] = seen + __popc(same);
            __syncwarp();
        }
        __syncthreads();
        if (threadIdx.x < kDigits) {   // per digit: over the warps, and the total to every block
            uint32_t t = 0;
            for (int w = 0; w < kClusterWarps; ++w) {
                const uint32_t here = sp.place[w][threadIdx.x];
                sp.place[w][threadIdx.x] = t;
                t += here;
            }
            for (int r = 0; r < kCluster; ++r) *cluster.map_shared_rank(&sp.totals[rank][threadIdx.x], r) = t;
        }
        cluster.sync();
        if (threadIdx.x < kDigits) {   // where this block's first item of a digit goes
            uint32_t total = 0, before = 0;
            for (int r = 0; r < kCluster; ++r) {
                const uint32_t t = sp.totals[r][threadIdx.x];
                if (r < rank) before += t;
                total += t;
            }
            uint32_t inc = total;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t up = __shfl_up_sync(0xFFFFFFFFu, inc, o);
                if (lane >= o) inc += up;
            }
            if (lane == 31) sp.scan[warp] = inc;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            for (int w = 0; w < warp; ++w) before += sp.scan[w];
            before += inc - total;
            for (int w = 0; w < kClusterWarps; ++w) sp.place[w][threadIdx.x] += before;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kMostPerBlock / kClusterThreads; ++r) {
            if (r >= rounds) break;
            const int i = warp * per_warp + r * 32 + lane;
            if (i >= mine) continue;
            const uint32_t to = sp.place[warp][(key[r] >> shift) & 0xFFu] + rank_in[r];
            const unsigned owner = to >> log_c, slot = (from ^ 1) * c + (to & (c - 1));
            *cluster.map_shared_rank(keys + slot, owner) = key[r];
            *cluster.map_shared_rank(order + slot, owner) = o_in[i];
        }
        cluster.sync();
    }
    next_may_start();
    for (int i = threadIdx.x; i < mine; i += kClusterThreads) {
        keys_out[base + i] = keys[from * c + i];
        order_out[base + i] = order[from * c + i];
    }
}

// ------------------------------------------------------------------------------------------------
// sums
// ------------------------------------------------------------------------------------------------

constexpr int kPiece = 32;   // sorted positions per piece
constexpr int kAhead = 8;    // rows of a piece that are on their way at a time (4 or 16, and pieces of 16 or 64, measured slower)

// A piece per blockDim.x threads (blockDim.y pieces per block), columns over blockDim.x and gridDim.y.
// partial: two rows of fp32 sums per piece -- slot 0 for a run that began in an earlier piece, slot 1 for one that begins
// here and goes on in the next.
template <int DT, int VEC>
__global__ void __launch_bounds__(kEmbedThreads) embed_sum_kernel(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ order,
                                                                  int64_t n, const void* __restrict__ dout, uint32_t vocab,
                                                                  int width, float scale, void* dweight, float* partial) {
    __shared__ uint32_t s_key[kMostRows][kPiece + 2];    // [piece of the block]; with the neighbours on both sides
    __shared__ uint32_t s_pos[kMostRows][kPiece];
    const int64_t piece = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y, first = piece * kPiece;
    uint32_t* const key = s_key[threadIdx.y];
    uint32_t* const pos = s_pos[threadIdx.y];
    after_previous();
    for (int i = threadIdx.x; i < kPiece + 2; i += blockDim.x) {
        const int64_t at = first + i - 1;
        key[i] = at >= 0 && at < n ? keys[at] : 0xFFFFFFFFu;   // larger than any key
        if (i >= 1 && i <= kPiece) pos[i - 1] = at < n ? order[at] : 0u;
    }
    __syncthreads();
    const int live = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(kPiece), n - first)));
    for (int c = (blockIdx.y * blockDim.x + threadIdx.x) * VEC; c < width; c += gridDim.y * blockDim.x * VEC) {
        float acc[VEC], f[VEC];
        bool begins = false;
        for (int p0 = 0; p0 < live && key[p0 + 1] < vocab; p0 += kAhead) {
            Bits<DT, VEC> b[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (p0 + k < live) b[k].load(dout, static_cast<int64_t>(pos[p0 + k]) * width + c);
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int p = p0 + k;
                if (p >= live) break;
                const uint32_t now = key[p + 1];
                if (now >= vocab) break;   // padding and tokens out of range: the last keys
                b[k].get(f);
                if (p == 0 || key[p] != now) {
                    begins = key[p] != now;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) acc[j] = f[j];
                } else {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) acc[j] += f[j];
                }
                if (p + 1 < live && key[p + 2] == now) continue;
                if (begins && key[p + 2] != now) {   // the run lies in this piece
#pragma unroll
                    for (int j = 0; j < VEC; ++j) f[j] = acc[j] * scale;
                    b[k].put(f);
                    b[k].store(dweight, static_cast<int64_t>(now) * width + c);
                } else {
                    float* const to = partial + (piece * 2 + (begins ? 1 : 0)) * width + c;
                    if constexpr (VEC % 4 == 0) {
#pragma unroll
                        for (int j = 0; j < VEC; j += 4)
                            *reinterpret_cast<float4*>(to + j) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
                    } else {
#pragma unroll
                        for (int j = 0; j < VEC; ++j) to[j] = acc[j];
                    }
                }
            }
        }
    }
    next_may_start();
}

// VEC sums of a partial row.
template <int VEC>
__device__ __forceinline__ void load_sums(const float* __restrict__ from, float (&f)[VEC]) {
    if constexpr (VEC % 4 == 0) {
#pragma unroll
        for (int j = 0; j < VEC; j += 4) {
            const float4 v = *reinterpret_cast<const float4*>(from + j);
            f[j] = v.x; f[j + 1] = v.y; f[j + 2] = v.z; f[j + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[j] = from[j];
    }
}

// The runs that span pieces: where a run begins, the partial sums of the pieces that it reaches are added up in order.  A
// warp per piece and slab of columns; a run over many pieces is left to the whole block, which sums sixteen slices of it
// side by side and then the slices in order.
constexpr int kJoinWarps = 16, kLongRun = 32;

// [first, last] of the pieces after `piece` that the run which begins in it and leaves it goes on in; false: no such run.
__device__ __forceinline__ bool run_from(const uint32_t* __restrict__ keys, int64_t n, uint32_t vocab, int64_t piece, uint32_t& key,
                                         int64_t& end) {
    const int64_t last = piece * kPiece + kPiece - 1;
    if (last + 1 >= n) return false;                                          // the last piece: nothing goes on
    key = keys[last];
    if (key >= vocab || keys[last + 1] != key) return false;
    // the run may fill the whole piece and come from an earlier one
    if (piece > 0 && keys[piece * kPiece] == key && keys[piece * kPiece - 1] == key) return false;
    // the last piece whose first key is the run's
    int64_t lo = piece + 1, hi = (n - 1) / kPiece;
    for (int64_t stride = 1; lo + stride <= hi; stride *= 2) {                // mostly the very next one
        if (keys[(lo + stride) * kPiece] != key) {
            hi = lo + stride - 1;
            break;
        }
        lo += stride;
    }
    while (lo < hi) {
        const int64_t mid = (lo + hi + 1) / 2;
        if (keys[mid * kPiece] == key) lo = mid; else hi = mid - 1;
    }
    end = lo;
    return true;
}

template <int DT, int VEC>
__global__ void __launch_bounds__(32 * kJoinWarps) embed_join_kernel(const uint32_t* __restrict__ keys, int64_t n, uint32_t vocab,
                                                                     int width, float scale, void* dweight,
                                                                     const float* __restrict__ partial) {
    __shared__ float s_sum[kJoinWarps][32][VEC + (VEC > 1 ? 1 : 0)];
    __shared__ int s_long;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t piece0 = static_cast<int64_t>(blockIdx.x) * kJoinWarps;
    if (threadIdx.x == 0) s_long = 0;
    after_previous();
    __syncthreads();
    const int c = (blockIdx.y * 32 + lane) * VEC;
    uint32_t key = 0;
    int64_t end = 0;
    const int64_t piece = piece0 + warp;
    const bool found = run_from(keys, n, vocab, piece, key, end);
    const bool long_run = found && end - piece > kLongRun;
    if (long_run && lane == 0) atomicOr(&s_long, 1 << warp);
    if (found && !long_run) {
        for (int at = c; at < width; at += gridDim.y * 32 * VEC) {
            float acc[VEC], f[VEC];
            load_sums<VEC>(partial + (piece * 2 + 1) * width + at, acc);
#pragma unroll 4
            for (int64_t q = piece + 1; q <= end; ++q) {
                load_sums<VEC>(partial + q * 2 * width + at, f);
#pragma unroll
                for (int j = 0; j < VEC; ++j) acc[j] += f[j];
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[j] *= scale;
            Bits<DT, VEC> b;
            b.put(acc);
            b.store(dweight, static_cast<int64_t>(key) * width + at);
        }
    }
    __syncthreads();
    for (int which = 0; which < kJoinWarps; ++which) {
        if (!(s_long >> which & 1)) continue;   // the same for the whole block
        run_from(keys, n, vocab, piece0 + which, key, end);
        const int64_t first = piece0 + which + 1, each = (end - first + 1 + kJoinWarps - 1) / kJoinWarps;
        const int64_t q0 = first + warp * each, q1 = min(q0 + each, end + 1);
        for (int base = blockIdx.y * 32 * VEC; base < width; base += gridDim.y * 32 * VEC) {
            const int at = base + lane * VEC;
            float acc[VEC], f[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
            if (at < width) {
                if (warp == 0) load_sums<VEC>(partial + ((piece0 + which) * 2 + 1) * width + at, acc);
#pragma unroll 8
                for (int64_t q = q0; q < q1; ++q) {
                    load_sums<VEC>(partial + q * 2 * width + at, f);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) acc[j] += f[j];
                }
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) s_sum[warp][lane][j] = acc[j];
            __syncthreads();
            if (warp == 0 && at < width) {
                for (int s = 1; s < kJoinWarps; ++s)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) acc[j] += s_sum[s][lane][j];
#pragma unroll
                for (int j = 0; j < VEC; ++j) acc[j] *= scale;
                Bits<DT, VEC> b;
                b.put(acc);
                b.store(dweight, static_cast<int64_t>(key) * width + at);
            }
            __syncthreads();
        }
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

// Threads across the pieces of a row (a power of two), the others over rows.
dim3 row_block(int pieces, int threads) {
    int x = 1;
    while (x < pieces && x < threads) x *= 2;
    const int y = threads / x;
    return dim3(x, y < kMostRows ? y : kMostRows);
}

template <int DT, int VEC>
int launch_sums(const uint32_t* keys, const uint32_t* order, int64_t n, const void* dout, int64_t vocab, int width, float scale,
                void* dweight, float* partial, cudaStream_t s) {
    const int64_t pieces = (n + kPiece - 1) / kPiece;
    dim3 block = row_block(width / VEC, kEmbedThreads);
    // pieces side by side in a warp take their turns at the ends of their runs: few pieces get blocks of their own
    while (block.y > 1 && pieces < 296ll * block.y) block.y /= 2;
    const int slabs = (width / VEC + block.x - 1) / block.x;
    const dim3 grid(static_cast<unsigned>((pieces + block.y - 1) / block.y), static_cast<unsigned>(slabs < 64 ? slabs : 64));
    cudaError_t e = launch_next(embed_sum_kernel<DT, VEC>, grid, block, s, keys, order, n, dout, static_cast<uint32_t>(vocab), width, scale,
                                dweight, partial);
    if (e == cudaSuccess && pieces > 1) {
        const int join_slabs = (width / VEC + 31) / 32;
        const dim3 join(static_cast<unsigned>((pieces + kJoinWarps - 1) / kJoinWarps),
                        static_cast<unsigned>(join_slabs < 64 ? join_slabs : 64));
        e = launch_next(embed_join_kernel<DT, VEC>, join, dim3(32 * kJoinWarps), s, keys, n, static_cast<uint32_t>(vocab), width, scale,
                        dweight, partial);
    }
    if (e != cudaSuccess) (void)cudaGetLastError();
    return record_cuda(e);
}

// Elements per access: 16 bytes, a word of two 16-bit elements, or one element -- what the width and the addresses allow.
int access_of(int dtype, int64_t width, const void* a, const void* b) {
    const int wide = dtype == ELX_F32 ? 4 : 8;
    if (width % wide == 0 && aligned(a, 16) && aligned(b, 16)) return wide;
    return dtype != ELX_F32 && width % 2 == 0 && aligned(a, 4) && aligned(b, 4) ? 2 : 1;
}

template <int DT, int VEC>
int launch_forward(const void* tokens, int index_bytes, int64_t n, const void* weight, int64_t vocab, int width, float scale,
                   void* out, cudaStream_t s) {
    // four accesses per thread, where the row is that wide
    const dim3 block = row_block((width / VEC + 3) / 4, kEmbedThreads);
    const int grid = grid_for((n + block.y - 1) / block.y, 16);
    if (grid < 0) return grid;
    if (index_bytes == 8) embed_forward_kernel<DT, VEC, int64_t><<<grid, block, 0, s>>>(tokens, n, weight, vocab, width, scale, out);
    else embed_forward_kernel<DT, VEC, int32_t><<<grid, block, 0, s>>>(tokens, n, weight, vocab, width, scale, out);
    return record_cuda(cudaGetLastError());
}

// Sort and zeros in one launch; for more tokens than a cluster's shared memory holds, in launches of their own.
int sort_tokens(const void* tokens, int index_bytes, int64_t n, int64_t vocab, int64_t padding, uint32_t* const (&keys)[2],
                uint32_t* const (&order)[2], uint32_t* counts, void* zeros, int64_t zero_bytes, int* result, cudaStream_t s) {
    int passes = 0;
    while (passes < 4 && (vocab >> (8 * passes)) != 0) ++passes;
    *result = 0;
    if (n <= kMostInCluster) {
        int log_c = 5;
        while ((static_cast<int64_t>(kCluster) << log_c) < n) ++log_c;
        const int smem = static_cast<int>(sizeof(SortSpace)) + (16 << log_c);
        constexpr int kMostSmem = static_cast<int>(sizeof(SortSpace)) + 16 * kMostPerBlock;
        static bool opted_in[64];
        int dev = -1;
        if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
            (void)cudaGetLastError();
            return ELX_ERR_NODEVICE;
        }
        if (!opted_in[dev]) {
            cudaError_t e = cudaFuncSetAttribute(embed_sort_kernel<int64_t>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem);
            if (e == cudaSuccess) e = cudaFuncSetAttribute(embed_sort_kernel<int32_t>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem);
            if (e != cudaSuccess) {
                const int rc = record_cuda(e);
                (void)cudaGetLastError();
                return rc;
            }
            opted_in[dev] = true;
        }
        // Clusters for the zeros: blocks with eight stores a thread, at most 15 of them (515 MB in 86 us and 161 MB in 33 us; with
        // as many as fit beside the sort 96 us and 31 us).
        const int64_t per_cluster = 32ll * kClusterThreads * 8 * kCluster, fill = (zero_bytes + per_cluster - 1) / per_cluster;
        const unsigned grid = kCluster * (1 + static_cast<unsigned>(fill < 1 ? 1 : fill > 15 ? 15 : fill));
        if (index_bytes == 8)
            embed_sort_kernel<int64_t><<<grid, kClusterThreads, smem, s>>>(tokens, n, vocab, padding, log_c, passes, keys[0], order[0],
                                                                          static_cast<char*>(zeros), zero_bytes);
        else
            embed_sort_kernel<int32_t><<<grid, kClusterThreads, smem, s>>>(tokens, n, vocab, padding, log_c, passes, keys[0], order[0],
                                                                          static_cast<char*>(zeros), zero_bytes);
        return record_cuda(cudaGetLastError());
    }
    const cudaError_t zeroed = cudaMemsetAsync(zeros, 0, zero_bytes, s);
    if (zeroed != cudaSuccess) return record_cuda(zeroed);
    const unsigned fill = static_cast<unsigned>((n + kSortThreads - 1) / kSortThreads);
    if (index_bytes == 8) embed_keys_kernel<int64_t><<<fill, kSortThreads, 0, s>>>(tokens, n, vocab, padding, keys[0], order[0]);
    else embed_keys_kernel<int32_t><<<fill, kSortThreads, 0, s>>>(tokens, n, vocab, padding, keys[0], order[0]);
    const unsigned tiles = static_cast<unsigned>((n + kSortTile - 1) / kSortTile);
    for (int pass = 0; pass < passes; ++pass, *result ^= 1) {
        const int from = *result, shift = 8 * pass;
        sort_count_kernel<<<tiles, kSortThreads, 0, s>>>(keys[from], n, shift, counts);
        sort_scan_kernel<<<1, 1024, 0, s>>>(counts, static_cast<int64_t>(tiles) * kDigits);
        sort_scatter_kernel<<<tiles, kSortThreads, 0, s>>>(keys[from], order[from], n, shift, counts, keys[from ^ 1], order[from ^ 1]);
    }
    return record_cuda(cudaGetLastError());
}

int check_embedding(const void* tokens, int index_bytes, int64_t n, int dtype, int64_t vocab, int64_t width, const void* a,
                    const void* b) {
    if (n < 0 || vocab <= 0 || width <= 0) return ELX_ERR_SIZE;
    if (n > 0 && !tokens) return ELX_ERR_NULL;
    if (!dtype_ok(dtype) || (index_bytes != 4 && index_bytes != 8)) return ELX_ERR_DTYPE;
    if (n > 0x7FFFFFFFll || vocab > 0x7FFFFFFFll || width > 0x3FFFFFFFll) return ELX_ERR_CAPACITY;
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
    const int w = static_cast<int>(width), access = access_of(dtype, width, weight, out);
#define ELX_FORWARD(DT, V) return launch_forward<DT, V>(tokens, index_bytes, n, weight, vocab, w, scale, out, s)
    if (dtype == ELX_F32) {
        if (access == 4) ELX_FORWARD(ELX_F32, 4);
        ELX_FORWARD(ELX_F32, 1);
    }
    if (dtype == ELX_F16) {
        if (access == 8) ELX_FORWARD(ELX_F16, 8);
        if (access == 2) ELX_FORWARD(ELX_F16, 2);
        ELX_FORWARD(ELX_F16, 1);
    }
    if (access == 8) ELX_FORWARD(ELX_BF16, 8);
    if (access == 2) ELX_FORWARD(ELX_BF16, 2);
    ELX_FORWARD(ELX_BF16, 1);
#undef ELX_FORWARD
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
    if (n == 0) {
        const cudaError_t zeroed = cudaMemsetAsync(dweight, 0, vocab * width * size, s);
        return record_cuda(zeroed);
    }
    char* at = static_cast<char*>(workspace);
    uint32_t *keys[2], *order[2];
    for (int k = 0; k < 2; ++k, at += 2 * space.keys) {
        keys[k] = reinterpret_cast<uint32_t*>(at);
        order[k] = reinterpret_cast<uint32_t*>(at + space.keys);
    }
    uint32_t* const counts = reinterpret_cast<uint32_t*>(at);
    float* const partial = reinterpret_cast<float*>(at + space.counts);
    int which = 0;
    const int sorted = sort_tokens(tokens, index_bytes, n, vocab, padding_idx, keys, order, counts, dweight, vocab * width * size,
                                   &which, s);
    if (sorted != ELX_OK) return sorted;
    const uint32_t *k = keys[which], *o = order[which];
    const int w = static_cast<int>(width), access = access_of(dtype, width, dout, dweight);
#define ELX_SUMS(DT, V) return launch_sums<DT, V>(k, o, n, dout, vocab, w, scale, dweight, partial, s)
    if (dtype == ELX_F32) {
        if (access == 4) ELX_SUMS(ELX_F32, 4);
        ELX_SUMS(ELX_F32, 1);
    }
    if (dtype == ELX_F16) {
        if (access == 8) ELX_SUMS(ELX_F16, 8);
        if (access == 2) ELX_SUMS(ELX_F16, 2);
        ELX_SUMS(ELX_F16, 1);
    }
    if (access == 8) ELX_SUMS(ELX_BF16, 8);
    if (access == 2) ELX_SUMS(ELX_BF16, 2);
    ELX_SUMS(ELX_BF16, 1);
#undef ELX_SUMS
}

}  // extern "C"
