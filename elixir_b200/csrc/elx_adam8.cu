// Part of the elixir_b200 CUDA library (C ABI: include/elixir_b200.h): the update with both moments in 8 bits, and
// the conversion of moments into that form and back.  The form itself: elx_moments.cuh.
#include "elx_adam_math.cuh"
#include "elx_common.cuh"
#include "elx_moments.cuh"

using namespace elx;

namespace {

__device__ __forceinline__ float sqrt_approx(float x) {
    float r;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// One element of the update.  The new moments are fp32 numbers with every product and sum rounded once (no fused
// multiply-add): their codes hang on the last bit, and so they are the same wherever the operation is restated.  The
// parameter's own step uses the unrounded (fp32) moments and approximate root and division: two relative errors of a
// few 2^-23 in a term that is lr times smaller than the parameter's own rounding allows to be seen.
__device__ __forceinline__ void adam8_elem(float& p, float& m, float& v, float g, const GroupK& k, int div_mode,
                                           float div, float inv_div) {
    if (div_mode == kMulInv) g *= inv_div;   // exact: the divisor is a power of two
    else if (div_mode == kTrueDiv) g = div_or_zero(g, div);
    g = fmaf(k.wd_l2, p, g);
    m = __fadd_rn(__fmul_rn(k.beta1, m), __fmul_rn(k.omb1, g));
    v = __fadd_rn(__fmul_rn(k.beta2, v), __fmul_rn(__fmul_rn(k.omb2, g), g));
    const float denom = sqrt_approx(v * k.rbc2) + k.eps;
    float upd = __fdividef(m * k.rbc1, denom);
    upd = fmaf(k.wd_w, p, upd);
    p = fmaf(-k.lr, upd, p);
}

struct Adam8Args {
    const ElxChunkDesc* descs;
    const ElxSeg* segs;
    const ElxHyper* hyper;
    ElxCtl* ctl;
    int first, count, n_groups;
    int64_t n_tiles;
};

constexpr int kAdam8Threads = 512;                     // one warp per block of a tile
static_assert(kAdam8Threads / 32 * kMomentBlock == kTile, "a tile is one block per warp");

// A tile is 16 blocks of 256 elements, one per warp; a lane owns 8 consecutive elements.  The block's exponent needs
// the largest magnitude of its new moments, which one redux instruction over the warp gives.
template <int DT>
__global__ void __launch_bounds__(kAdam8Threads, 2) adam8_kernel(const Adam8Args a) {
    using T = typename Lp<DT>::T;
    __shared__ GroupK s_group[kMaxGroups];
    __shared__ ChunkCursor s_cur;
    __shared__ SegCursor s_seg;
    ElxCtl* ctl = a.ctl;
    const bool skip = ctl->skip != 0;
    const float div = ctl->div_scale, inv_div = ctl->inv_div;
    const int div_mode = div > 0.0f ? (inv_div != 0.0f ? kMulInv : kTrueDiv) : kNoDiv;
    const int step = ctl->step;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (!skip)
        for (int gi = threadIdx.x; gi < a.n_groups; gi += blockDim.x) s_group[gi] = derive_group(a.hyper[gi], step);
    if (threadIdx.x == 0) {
        s_seg.b = s_seg.e = 0;
        s_seg.group = -1;
        s_seg.chunk = -1;
    }
    cursor_reset(s_cur);

    const int64_t tile_lo = a.descs[a.first].tile_begin;
    float nan_acc = 0.0f;
    bool bad_desc = false;
    for (int64_t it = blockIdx.x; it < a.n_tiles; it += gridDim.x) {
        const int64_t t = tile_lo + it;
        if (!locate_chunk(a.descs, a.first, a.count, t, s_cur) || s_cur.d.dtype != DT) {
            bad_desc = true;
            continue;
        }
        const int64_t n = s_cur.d.n_shard;
        const int64_t e0 = (t - s_cur.t0) * kTile;
        const int64_t e1 = min(e0 + kTile, n);
        const ElxSeg* csegs = a.segs + s_cur.d.seg_first;
        const int n_segs = s_cur.d.seg_count;
        if (s_seg.chunk != s_cur.index || e0 < s_seg.b || e0 >= s_seg.e) {
            __syncthreads();
            if (threadIdx.x == 0) {
                const int si = find_seg(csegs, n_segs, e0);
                s_seg.chunk = s_cur.index;
                s_seg.b = si >= 0 ? csegs[si].begin : 0;
                s_seg.e = si >= 0 ? csegs[si].end : 0;
                s_seg.group = si >= 0 ? csegs[si].group : -1;
            }
            __syncthreads();
        }
        const int grp = s_seg.group;
        const bool one_group = s_seg.b <= e0 && e1 <= s_seg.e && grp >= 0 && grp < a.n_groups;
        float* const master = s_cur.d.master;
        T* const lowp = static_cast<T*>(s_cur.d.grad_param);
        const T* const gsrc = static_cast<const T*>(grad_source(s_cur.d));
        uint8_t* const state_m = reinterpret_cast<uint8_t*>(s_cur.d.exp_avg);
        uint8_t* const state_v = reinterpret_cast<uint8_t*>(s_cur.d.exp_avg_sq);
        uint8_t* const exps_m = state_m + moment_exps_at(n);
        uint8_t* const exps_v = state_v + moment_exps_at(n);
        const int64_t b0 = e0 + warp * kMomentBlock;   // first element of the warp's block
        if (b0 >= e1) continue;
        const int64_t block = b0 / kMomentBlock;

        if (!skip && e1 - e0 == kTile && s_cur.vec_ok && one_group) {
            const GroupK k = s_group[grp];
            const int64_t e = b0 + lane * 8;
            float g[8], p[8];
            load_lowp<DT, 8>(gsrc, e0, g);
            load_f32<8>(master, e0, p);
            const uint2 cm = *reinterpret_cast<const uint2*>(state_m + e), cv = *reinterpret_cast<const uint2*>(state_v + e);
            const float sm = decode_scale(exps_m[block]), sv = decode_scale(exps_v[block]);
            float m[8], v[8];
            uint32_t top_m = 0, top_v = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                m[j] = decode<FirstMoment>(((j < 4 ? cm.x : cm.y) >> (8 * (j & 3))) & 0xFFu, sm);
                v[j] = decode<SecondMoment>(((j < 4 ? cv.x : cv.y) >> (8 * (j & 3))) & 0xFFu, sv);
                nan_acc = fmaf(0.0f, g[j], nan_acc);
                adam8_elem(p[j], m[j], v[j], g[j], k, div_mode, div, inv_div);
                top_m = max(top_m, __float_as_uint(m[j]) & 0x7FFFFFFFu);
                top_v = max(top_v, __float_as_uint(v[j]) & 0x7FFFFFFFu);
            }
            const uint32_t em = block_exponent(__reduce_max_sync(0xFFFFFFFFu, top_m));
            const uint32_t ev = block_exponent(__reduce_max_sync(0xFFFFFFFFu, top_v));
            const float xm = encode_scale(em), xv = encode_scale(ev);
            const uint32_t key = dither_key(step, s_cur.index, block);
            uint2 om = make_uint2(0, 0), ov = make_uint2(0, 0);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t r = dither_bits(key, lane * 8 + j);
                const uint32_t a0 = encode<FirstMoment>(m[j], xm, (r & 0xFFFFu) << 4) << (8 * (j & 3));
                const uint32_t a1 = encode<SecondMoment>(v[j], xv, (r >> 16) << 4) << (8 * (j & 3));
                if (j < 4) { om.x |= a0; ov.x |= a1; } else { om.y |= a0; ov.y |= a1; }
            }
            store_f32<8>(master, e0, p);
            store_lowp<DT, 8>(lowp, e0, p);
            *reinterpret_cast<uint2*>(state_m + e) = om;
            *reinterpret_cast<uint2*>(state_v + e) = ov;
            if (lane == 0) {
                exps_m[block] = static_cast<uint8_t>(em);
                exps_v[block] = static_cast<uint8_t>(ev);
            }
            continue;
        }

        // Skipped step, shard tail, segment boundary, uncovered elements or unaligned pointers: one element at a time.
        // An uncovered element of a block that is updated keeps the values of its moments, under the block's new scale.
        const int64_t b1 = min(b0 + kMomentBlock, e1);
        const bool touched = !skip && !range_uncovered(csegs, n_segs, b0, b1, s_cur.d.n_valid);
        float m[8], v[8];
        uint32_t top_m = 0, top_v = 0;
        const float sm = touched ? decode_scale(exps_m[block]) : 0.0f, sv = touched ? decode_scale(exps_v[block]) : 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            m[j] = v[j] = 0.0f;
            const int64_t e = b0 + lane + 32 * j;
            if (e >= b1) continue;
            float p = master[e];
            if (touched) {
                m[j] = decode<FirstMoment>(state_m[e], sm);
                v[j] = decode<SecondMoment>(state_v[e], sv);
                const int si = find_seg(csegs, n_segs, e);
                const int ge = si >= 0 && e < csegs[si].end ? csegs[si].group : -1;
                if (ge >= 0 && ge < a.n_groups) {
                    const float g = Lp<DT>::to_float(gsrc[e]);
                    nan_acc = fmaf(0.0f, g, nan_acc);
                    adam8_elem(p, m[j], v[j], g, s_group[ge], div_mode, div, inv_div);
                    master[e] = p;
                }
                top_m = max(top_m, __float_as_uint(m[j]) & 0x7FFFFFFFu);
                top_v = max(top_v, __float_as_uint(v[j]) & 0x7FFFFFFFu);
            }
            lowp[e] = Lp<DT>::from_float(p);
        }
        if (!touched) continue;   // the whole warp: one block, one decision
        const uint32_t em = block_exponent(__reduce_max_sync(0xFFFFFFFFu, top_m));
        const uint32_t ev = block_exponent(__reduce_max_sync(0xFFFFFFFFu, top_v));
        const float xm = encode_scale(em), xv = encode_scale(ev);
        const uint32_t key = dither_key(step, s_cur.index, block);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t e = b0 + lane + 32 * j;
            if (e >= b1) continue;
            const uint32_t r = dither_bits(key, lane + 32 * j);
            state_m[e] = static_cast<uint8_t>(encode<FirstMoment>(m[j], xm, (r & 0xFFFFu) << 4));
            state_v[e] = static_cast<uint8_t>(encode<SecondMoment>(v[j], xv, (r >> 16) << 4));
        }
        if (lane == 0) {
            exps_m[block] = static_cast<uint8_t>(em);
            exps_v[block] = static_cast<uint8_t>(ev);
        }
    }

    const unsigned late = __ballot_sync(0xFFFFFFFFu, nan_acc != nan_acc);
    const unsigned bad = __ballot_sync(0xFFFFFFFFu, bad_desc);
    if (lane == 0) {
        if (late) {
            atomicOr(&ctl->late_inf, 1u);
            atomicOr(&ctl->status, ELX_STAT_LATE_INF);
        }
        if (bad) atomicOr(&ctl->status, ELX_STAT_BAD_DESC);
    }
}

template <int DT>
int launch_adam8(const Adam8Args& a, cudaStream_t s) {
    static const int resident = resident_ctas(adam8_kernel<DT>, kAdam8Threads);
    const int grid = grid_for(a.n_tiles, resident);
    if (grid < 0) return grid;
    adam8_kernel<DT><<<grid, kAdam8Threads, 0, s>>>(a);
    return record_cuda(cudaGetLastError());
}

// ------------------------------------------------------------------------------------------------
// conversion
// ------------------------------------------------------------------------------------------------

constexpr int kConvThreads = 256;

// One warp per block and moment array; the two moments of a block one after the other.
template <class M>
__device__ __forceinline__ void pack_block(const float* __restrict__ x, uint8_t* state, int64_t n, int64_t block, bool vec) {
    const int lane = threadIdx.x & 31;
    const int64_t b0 = block * kMomentBlock;
    const bool whole = vec && b0 + kMomentBlock <= n;
    float f[8];
    uint32_t top = 0;
    if (whole) {
        const U8 r = ld256(x + b0 + lane * 8);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = __uint_as_float(r.x[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t e = b0 + lane * 8 + j;
            f[j] = e < n ? x[e] : 0.0f;
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(f[j]) & 0x7FFFFFFFu);
    const uint32_t exp = block_exponent(__reduce_max_sync(0xFFFFFFFFu, top));
    const float scale = encode_scale(exp);
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j / 4] |= encode<M>(f[j], scale, kRoundNearest) << (8 * (j & 3));
    if (whole) {
        *reinterpret_cast<uint2*>(state + b0 + lane * 8) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t e = b0 + lane * 8 + j;
            if (e < n) state[e] = static_cast<uint8_t>(w[j / 4] >> (8 * (j & 3)));
        }
    }
    if (lane == 0) state[moment_exps_at(n) + block] = static_cast<uint8_t>(exp);
}

__global__ void __launch_bounds__(kConvThreads) pack_kernel(const float* __restrict__ m, const float* __restrict__ v, int64_t n,
                                                            uint8_t* state_m, uint8_t* state_v, int vec) {
    const int64_t blocks = moment_blocks(n);
    const int64_t stride = static_cast<int64_t>(gridDim.x) * (kConvThreads / 32);
    for (int64_t b = blockIdx.x * (kConvThreads / 32) + (threadIdx.x >> 5); b < blocks; b += stride) {
        pack_block<FirstMoment>(m, state_m, n, b, vec);
        pack_block<SecondMoment>(v, state_v, n, b, vec);
    }
}

template <class M, int DT>
__device__ __forceinline__ void unpack_block(const uint8_t* __restrict__ state, void* out, int64_t n, int64_t block, bool vec) {
    using T = typename Lp<DT>::T;
    const int lane = threadIdx.x & 31;
    const int64_t e0 = block * kMomentBlock + lane * 8;
    const float scale = decode_scale(state[moment_exps_at(n) + block]);
    T* const o = static_cast<T*>(out);
    if (vec && (block + 1) * kMomentBlock <= n) {
        const uint2 c = *reinterpret_cast<const uint2*>(state + e0);
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = decode<M>(((j < 4 ? c.x : c.y) >> (8 * (j & 3))) & 0xFFu, scale);
        if constexpr (DT == ELX_F32) {
            U8 r;
#pragma unroll
            for (int j = 0; j < 8; ++j) r.x[j] = __float_as_uint(f[j]);
            st256(o + e0, r);
        } else {
            U4 r;
#pragma unroll
            for (int j = 0; j < 4; ++j) r.x[j] = Lp<DT>::pack2(f[2 * j], f[2 * j + 1]);
            st128(o + e0, r);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (e0 + j < n) o[e0 + j] = Lp<DT>::from_float(decode<M>(state[e0 + j], scale));
    }
}

template <int DT>
__global__ void __launch_bounds__(kConvThreads) unpack_kernel(const uint8_t* __restrict__ state_m, const uint8_t* __restrict__ state_v,
                                                              int64_t n, void* m, void* v, int vec) {
    const int64_t blocks = moment_blocks(n);
    const int64_t stride = static_cast<int64_t>(gridDim.x) * (kConvThreads / 32);
    for (int64_t b = blockIdx.x * (kConvThreads / 32) + (threadIdx.x >> 5); b < blocks; b += stride) {
        unpack_block<FirstMoment, DT>(state_m, m, n, b, vec);
        unpack_block<SecondMoment, DT>(state_v, v, n, b, vec);
    }
}

}  // namespace

extern "C" {

int64_t elx_moment_state_bytes(int64_t n) { return n < 0 ? ELX_ERR_SIZE : moment_state_bytes(n); }

int elx_adam8_multi(const ElxChunkDesc* descs, int first, int count, int64_t n_tiles, int dtype, const ElxSeg* segs,
                    const ElxHyper* hyper, int n_groups, ElxCtl* ctl, void* stream) {
    if (!descs || !ctl) return ELX_ERR_NULL;
    if (n_groups > 0 && (!segs || !hyper)) return ELX_ERR_NULL;
    if (!dtype_ok(dtype)) return ELX_ERR_DTYPE;
    if (first < 0 || count < 0 || n_tiles < 0 || n_groups < 0) return ELX_ERR_SIZE;
    if (n_groups > kMaxGroups) return ELX_ERR_CAPACITY;
    if (!aligned(descs, 8) || !aligned(ctl, 16) || (segs && !aligned(segs, 8)) || (hyper && !aligned(hyper, 4)))
        return ELX_ERR_ALIGN;
    if (count == 0 || n_tiles == 0) return ELX_OK;
    const Adam8Args a = {descs, segs, hyper, ctl, first, count, n_groups, n_tiles};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case ELX_F16: return launch_adam8<ELX_F16>(a, s);
        case ELX_BF16: return launch_adam8<ELX_BF16>(a, s);
    }
    return launch_adam8<ELX_F32>(a, s);
}

int elx_moments_pack(const float* exp_avg, const float* exp_avg_sq, int64_t n, void* state_m, void* state_v, void* stream) {
    if (!exp_avg || !exp_avg_sq || !state_m || !state_v) return ELX_ERR_NULL;
    if (n < 0) return ELX_ERR_SIZE;
    if (!aligned(exp_avg, 4) || !aligned(exp_avg_sq, 4)) return ELX_ERR_ALIGN;
    if (n == 0) return ELX_OK;
    const int vec = aligned(exp_avg, 32) && aligned(exp_avg_sq, 32) && aligned(state_m, 8) && aligned(state_v, 8);
    const int grid = grid_for((moment_blocks(n) + kConvThreads / 32 - 1) / (kConvThreads / 32), 8);
    if (grid < 0) return grid;
    pack_kernel<<<grid, kConvThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        exp_avg, exp_avg_sq, n, static_cast<uint8_t*>(state_m), static_cast<uint8_t*>(state_v), vec);
    return record_cuda(cudaGetLastError());
}

int elx_moments_unpack(const void* state_m, const void* state_v, int64_t n, int dtype, void* exp_avg, void* exp_avg_sq,
                       void* stream) {
    if (!state_m || !state_v || !exp_avg || !exp_avg_sq) return ELX_ERR_NULL;
    if (dtype != ELX_F32 && dtype != ELX_BF16) return ELX_ERR_DTYPE;
    if (n < 0) return ELX_ERR_SIZE;
    if (!aligned(exp_avg, dtype_bytes(dtype)) || !aligned(exp_avg_sq, dtype_bytes(dtype))) return ELX_ERR_ALIGN;
    if (n == 0) return ELX_OK;
    const int vec = aligned(exp_avg, 32) && aligned(exp_avg_sq, 32) && aligned(state_m, 8) && aligned(state_v, 8);
    const int grid = grid_for((moment_blocks(n) + kConvThreads / 32 - 1) / (kConvThreads / 32), 8);
    if (grid < 0) return grid;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const uint8_t *sm = static_cast<const uint8_t*>(state_m), *sv = static_cast<const uint8_t*>(state_v);
    if (dtype == ELX_F32) unpack_kernel<ELX_F32><<<grid, kConvThreads, 0, s>>>(sm, sv, n, exp_avg, exp_avg_sq, vec);
    else unpack_kernel<ELX_BF16><<<grid, kConvThreads, 0, s>>>(sm, sv, n, exp_avg, exp_avg_sq, vec);
    return record_cuda(cudaGetLastError());
}

}  // extern "C"
