// Part of the elixir_b200 CUDA library (C ABI: include/elixir_b200.h): the update with both moments in 8 bits, and
// the conversion of moments into that form and back.  The form itself: elx_moments.cuh.
#include "elx_adam_math.cuh"
#include "elx_common.cuh"
#include "elx_moments.cuh"

using namespace elx;

namespace {

// ------------------------------------------------------------------------------------------------
// one element
// ------------------------------------------------------------------------------------------------

// What the update needs of a parameter group beside GroupK, with powers of two folded in: the second moment is scaled
// by 2^24 before its root, so that its smallest subnormal is a normal number there and the flushing forms of root and
// reciprocal (one instruction each) lose nothing; 2^12 then stands in eps and in the first moment's factor as well.
struct Group8 {
    float lr, beta1, omb1, beta2, omb2, wd_l2, wd_w;
    float rbc1, rbc2, eps;   // 2^12 / bc1, 2^24 / bc2, 2^12 eps
    float one;               // 1 (see new_moments2)
};

// By two threads per group, a moment each: the powers in double are most of a small launch's start.
__device__ __noinline__ void derive_half(const ElxHyper& h, int step, int second, Group8& k) {
    const float beta = second ? h.beta2 : h.beta1;
    const double bc = h.bias_correction ? 1.0 - pow(static_cast<double>(beta), static_cast<double>(step)) : 1.0;
    const float rbc = static_cast<float>(1.0 / bc);
    if (second) {
        k.beta2 = beta;
        k.omb2 = 1.0f - beta;
        k.rbc2 = rbc * 16777216.0f;
        k.wd_l2 = h.adamw_mode ? 0.0f : h.weight_decay;
        k.wd_w = h.adamw_mode ? h.weight_decay : 0.0f;
    } else {
        k.beta1 = beta;
        k.omb1 = 1.0f - beta;
        k.rbc1 = rbc * 4096.0f;
        k.lr = h.lr;
        k.one = 1.0f;
        k.eps = h.eps * 4096.0f;
    }
}

__device__ __forceinline__ float unscale(float g, int div_mode, float div, float inv_div) {
    if (div_mode == kMulInv) return g * inv_div;   // exact: the divisor is a power of two
    return div_mode == kTrueDiv ? div_or_zero(g, div) : g;
}

// The new moments: fp32 numbers with every product and sum rounded once, no fused multiply-add.  Which code they get
// hangs on their last bit, and so it is the same wherever the operation is restated.
__device__ __forceinline__ void new_moments(float p, float& m, float& v, float g, const Group8& k) {
    if (k.wd_l2 != 0.0f) g = fmaf(k.wd_l2, p, g);   // uniform: one group per call site's block, or the element-wise path
    m = __fadd_rn(__fmul_rn(k.beta1, m), __fmul_rn(k.omb1, g));
    v = __fadd_rn(__fmul_rn(k.beta2, v), __fmul_rn(__fmul_rn(k.omb2, g), g));
}

// The parameter's step, by the unrounded (fp32) moments: approximate root and reciprocal, off by a few 2^-23 in a term
// that is lr times smaller than what the parameter's own rounding allows to be seen.  For second moments below 2^31.
__device__ __forceinline__ float new_param(float p, float m, float v, const Group8& k) {
    float root, inv;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(root) : "f"(v * k.rbc2));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(root + k.eps));
    return fmaf(-k.lr, fmaf(k.wd_w, p, __fmul_rn(__fmul_rn(m, k.rbc1), inv)), p);
}
// The same for moments of any size.
__device__ __noinline__ float new_param_wide(float p, float m, float v, const Group8& k) {
    const float root = sqrtf(v * (k.rbc2 * 0x1p-24f)) * 4096.0f;
    return fmaf(-k.lr, fmaf(k.wd_w, p, m * k.rbc1 / (root + k.eps)), p);
}

// Exponent bytes up to which one product decodes or encodes (2^(E - 15), 2^(15 - E) and, for the second moment,
// 2^(E - 31), 2^(31 - E) are normal numbers): first moments below 2^15, second moments below 2^31.  Others, and blocks
// that are not finite, take the element-wise path.
constexpr uint32_t kEasyM = 141, kEasyV = 157;

// ------------------------------------------------------------------------------------------------
// one block of 256 elements by one warp, element by element
// ------------------------------------------------------------------------------------------------

struct BlockAt {
    float* p;              // first element of the block in each array: shared or global memory
    const void* g;
    void* lowp;            // may be g itself
    uint8_t *cm, *cv;
    uint8_t *em, *ev;
    int64_t e0;            // its index in the shard
    int len;
    const ElxSeg* segs;
    int seg_lo, seg_hi;    // the segments that may reach into the block: [seg_lo, seg_hi]
    int group;             // group of the whole block, or -1: by the segments
};

// The segments that reach into elements [b0, b1) of a shard, searched from segment `from` on (the last one that begins
// at or before an earlier element, or -1).  false: none does.  group: that of a segment which covers all of them, or -1.
__device__ __forceinline__ bool block_segments(const ElxSeg* __restrict__ segs, int n_segs, int from, int n_groups, int64_t b0, int64_t b1,
                                               int& lo, int& hi, int& group) {
    lo = max(from, 0);
    group = -1;
    while (lo < n_segs && segs[lo].end <= b0) ++lo;      // a tile's segments lie close together
    if (lo >= n_segs || segs[lo].begin >= b1) return false;
    hi = lo;
    while (hi + 1 < n_segs && segs[hi + 1].begin < b1) ++hi;
    if (segs[lo].begin <= b0 && segs[lo].end >= b1 && segs[lo].group < n_groups) group = segs[lo].group;
    return true;
}

// Shard tail, segment boundary, uncovered elements, unaligned arrays, moments of extreme size.  An uncovered element of
// a block that is updated keeps the values of its moments, under the block's new scale.
template <int DT>
__device__ __noinline__ void update_block(const BlockAt& b, const Group8* s_group, int n_groups, uint32_t key, int div_mode,
                                          float div, float inv_div, float& nan_acc) {
    using T = typename Lp<DT>::T;
    const int lane = threadIdx.x & 31;
    const uint32_t em0 = *b.em, ev0 = *b.ev;
    const float sm = decode_scale(em0), sv = decode_scale(ev0);
    float m[8], v[8], p[8];
    int grp[8];
    uint32_t top_m = 0, top_v = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) grp[j] = b.group;
    if (b.group < 0) {
        for (int si = b.seg_lo; si <= b.seg_hi; ++si) {
            const ElxSeg seg = b.segs[si];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int64_t e = b.e0 + lane + 32 * j;
                if (e >= seg.begin && e < seg.end) grp[j] = seg.group;
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int i = lane + 32 * j;
        m[j] = v[j] = p[j] = 0.0f;
        if (i >= b.len) continue;
        p[j] = b.p[i];
        m[j] = decode<FirstMoment>(b.cm[i], sm);
        v[j] = decode<SecondMoment>(b.cv[i], sv);
        if (grp[j] >= 0 && grp[j] < n_groups) {
            const float g = Lp<DT>::to_float(static_cast<const T*>(b.g)[i]);
            nan_acc = fmaf(0.0f, g, nan_acc);
            new_moments(p[j], m[j], v[j], unscale(g, div_mode, div, inv_div), s_group[grp[j]]);
        } else {
            grp[j] = -1;
        }
        top_m = max(top_m, __float_as_uint(m[j]) & 0x7FFFFFFFu);
        top_v = max(top_v, __float_as_uint(v[j]) & 0x7FFFFFFFu);
    }
    const uint32_t em = block_exponent(__reduce_max_sync(0xFFFFFFFFu, top_m));
    const uint32_t ev = block_exponent(__reduce_max_sync(0xFFFFFFFFu, top_v));
    // A block that is not finite, whatever made it so: a finite gradient whose square passes fp32's range does, and so does a
    // block that was not before.  All 256 elements of it are lost, which is reported like a gradient that is not finite.
    if (max(em, ev) == 255u) nan_acc = __uint_as_float(0x7FC00000u);
    const float xm = encode_scale(em), xv = encode_scale(ev);
    const bool easy = em <= kEasyM && ev <= kEasyV;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int i = lane + 32 * j;
        if (i >= b.len) continue;
        const uint32_t r = dither_bits(key, i);
        b.cm[i] = static_cast<uint8_t>(encode<FirstMoment>(m[j], xm, (r & 0xFFFFu) << 4));
        b.cv[i] = static_cast<uint8_t>(encode<SecondMoment>(v[j], xv, (r >> 16) << 4));
        if (grp[j] >= 0) {
            const Group8& k = s_group[grp[j]];
            p[j] = easy ? new_param(p[j], m[j], v[j], k) : new_param_wide(p[j], m[j], v[j], k);
            b.p[i] = p[j];
        }
        static_cast<T*>(b.lowp)[i] = Lp<DT>::from_float(p[j]);
    }
    if (lane == 0) {
        *b.em = static_cast<uint8_t>(em);
        *b.ev = static_cast<uint8_t>(ev);
    }
}

// Byte j of a word moved to the top of a word, and the top bytes of four words as one word.
__device__ __forceinline__ uint32_t byte_to_top(uint32_t w, int j) { return __byte_perm(w, 0, 0x0444 | (j << 12)); }
__device__ __forceinline__ uint32_t top_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410);
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Two elements per instruction: the packed fp32 operations take one issue slot for both, and issue slots are what the
// update runs short of first.  The same roundings as new_moments() and new_param().
// A sum of two products is written as a fused multiply-add of the one product with a 1 that the compiler cannot see
// through: CUDA 12.9 fuses mul.rn.f32x2 with a following add.rn.f32x2 (as it does the intrinsics for them), which changes
// the last bit of a moment.
__device__ __forceinline__ void new_moments2(float2 p, float2& m, float2& v, float2 g, const Group8& k, bool l2) {
    if (l2) g = fma2(both(k.wd_l2), p, g);
    m = fma2(mul2(both(k.beta1), m), both(k.one), mul2(both(k.omb1), g));
    v = fma2(mul2(both(k.beta2), v), both(k.one), mul2(mul2(both(k.omb2), g), g));
}
__device__ __forceinline__ float2 new_param2(float2 p, float2 m, float2 v, const Group8& k) {
    const float2 vh = mul2(v, both(k.rbc2));
    float2 root, inv;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(root.x) : "f"(vh.x));
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(root.y) : "f"(vh.y));
    const float2 den = add2(root, both(k.eps));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv.x) : "f"(den.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv.y) : "f"(den.y));
    const float2 upd = fma2(both(k.wd_w), p, mul2(mul2(m, both(k.rbc1)), inv));
    return fma2(both(-k.lr), upd, p);
}

// ------------------------------------------------------------------------------------------------
// the kernel
// ------------------------------------------------------------------------------------------------
//
// Tiles of 4096 elements stream through a ring of stages in shared memory (cp.async.bulk in, cp.async.bulk out,
// completion by mbarriers), as in the fp32 form of the update: one CTA per SM, 16 computing warps and one warp whose
// first lane moves the data.  A stage is 32 KB with 16-bit gradients (8 g, 16 p, 4 + 4 codes) plus the 16 + 16 exponent
// bytes of its 16 blocks, so six stages fit.  A warp owns one block of 256 elements of every tile: the block's exponent
// needs the largest of its new moments, which stay in registers, and one redux instruction per moment gives it.  So no
// computing warp ever waits for another; each tells the mover by itself that its part of the stage is done.
//
// The bytes bound it (16 per element of 16-bit chunks): 8 x 32 Mi elements take 732 us, 5.87 TB/s, against 1253 us and
// 5.98 TB/s for the update with fp32 moments, and 6.4 TB/s for a plain copy.  The arithmetic takes about 60 instructions per
// element and so 60 % of the issue slots; packed fp32 operations, scales folded into one product, codes kept in the top byte
// of a word and all that is rare (huge or non-finite moments, block borders) left to update_block() keep it there.  One
// launch of three small shards takes 8 us, most of it the first tile's way through the ring.
struct Adam8Args {
    const ElxChunkDesc* descs;
    const ElxSeg* segs;
    const ElxHyper* hyper;
    ElxCtl* ctl;
    int first, count, n_groups;
    int64_t n_tiles;
};

constexpr int kWarps = kTile / kMomentBlock;   // 16 computing warps, a block of the tile each
constexpr int kComputing = 32 * kWarps;
constexpr int kThreads = kComputing + 32;
constexpr int kBatch = 16;                     // tiles the mover's lanes look up at a time

template <int DT>
struct Stage8 {
    static constexpr int kP = 0;
    static constexpr int kG = 4 * kTile;
    static constexpr int kGBytes = kTile * Lp<DT>::kBytes;
    static constexpr int kM = kG + kGBytes;
    static constexpr int kV = kM + kTile;
    static constexpr int kEm = kV + kTile;
    static constexpr int kEv = kEm + kWarps;
    static constexpr int kLoaded = kEv + kWarps;
    static constexpr int kBytes = (kLoaded + 127) / 128 * 128;
    static constexpr int kStages = DT == ELX_F32 ? 5 : 6;
};

// kWhole: a whole tile inside one segment.  kMixed: a whole tile that segments cover in part or by several groups; it
// goes through the ring all the same and each warp looks its block up.  kRefresh: a whole tile that gets only its working
// copy (no segment reaches it, or the step is skipped).  kRagged: the end of a shard, or unaligned arrays; worked on in
// place in global memory.
enum { kBad = 0, kWhole = 1, kMixed = 2, kRefresh = 3, kRagged = 4 };

struct Slot8 {
    float* master;
    void* lowp;
    const void* gsrc;
    uint8_t *state_m, *state_v, *exps_m, *exps_v;
    const ElxSeg* segs;
    int64_t e0, e1;
    int n_segs, seg, group, kind, chunk;   // seg: the last segment that begins at or before e0, or -1
};

// The mover's view of the table: the descriptor and the segment it is in.
struct Cursor8 {
    int64_t t0 = 0, t1 = 0;
    int index = -1;
    bool vec_ok = false;
    ElxChunkDesc d;
    int64_t seg_b = 0, seg_e = 0;
    int seg = -1, seg_group = -1;
};

template <int DT>
__device__ __forceinline__ void classify(const Adam8Args& a, int64_t t, bool skip, Cursor8& c, Slot8& out) {
    if (!(t >= c.t0 && t < c.t1)) {
        int lo = a.first, hi = a.first + a.count - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (a.descs[mid].tile_begin <= t) lo = mid; else hi = mid - 1;
        }
        c.d = a.descs[lo];
        c.index = lo;
        c.t0 = c.d.tile_begin;
        c.t1 = c.t0 + tiles_of(c.d.n_shard);
        c.seg_b = c.seg_e = 0;
        const uintptr_t bits = reinterpret_cast<uintptr_t>(c.d.master) | reinterpret_cast<uintptr_t>(c.d.exp_avg) |
                               reinterpret_cast<uintptr_t>(c.d.exp_avg_sq) | reinterpret_cast<uintptr_t>(c.d.grad_param) |
                               reinterpret_cast<uintptr_t>(c.d.grad_src);
        c.vec_ok = (bits & 15u) == 0;
    }
    if (!(t >= c.t0 && t < c.t1) || c.d.dtype != DT) {
        out.kind = kBad;
        return;
    }
    out.e0 = (t - c.t0) * kTile;
    out.e1 = min(out.e0 + kTile, c.d.n_shard);
    out.segs = a.segs + c.d.seg_first;
    out.n_segs = c.d.seg_count;
    if (out.e0 < c.seg_b || out.e0 >= c.seg_e) {
        c.seg = find_seg(out.segs, out.n_segs, out.e0);
        c.seg_b = c.seg >= 0 ? out.segs[c.seg].begin : 0;
        c.seg_e = c.seg >= 0 ? out.segs[c.seg].end : 0;
        c.seg_group = c.seg >= 0 ? out.segs[c.seg].group : -1;
    }
    out.seg = c.seg;
    const bool one = c.seg_b <= out.e0 && out.e1 <= c.seg_e && c.seg_group >= 0 && c.seg_group < a.n_groups;
    out.group = one ? c.seg_group : -1;
    out.master = c.d.master;
    out.lowp = c.d.grad_param;
    out.gsrc = grad_source(c.d);
    out.state_m = reinterpret_cast<uint8_t*>(c.d.exp_avg);
    out.state_v = reinterpret_cast<uint8_t*>(c.d.exp_avg_sq);
    out.exps_m = out.state_m + moment_exps_at(c.d.n_shard);
    out.exps_v = out.state_v + moment_exps_at(c.d.n_shard);
    out.chunk = c.index;
    const bool whole = out.e1 - out.e0 == kTile && c.vec_ok;
    if (!whole) out.kind = kRagged;
    else if (skip) out.kind = kRefresh;
    else if (one) out.kind = kWhole;
    else out.kind = range_uncovered(out.segs, out.n_segs, out.e0, out.e1, c.d.n_valid) ? kRefresh : kMixed;
}

template <int DT>
__global__ void __launch_bounds__(kThreads, 1) adam8_kernel(const __grid_constant__ Adam8Args a) {
    using S = Stage8<DT>;
    using T = typename Lp<DT>::T;
    constexpr int kStages = S::kStages;
    extern __shared__ __align__(128) unsigned char s_dyn[];
    __shared__ Group8 s_group[kMaxGroups];
    __shared__ Slot8 s_slot[2 * kBatch];
    __shared__ uint32_t s_key[2 * kBatch][kWarps];      // dither keys of the tiles' blocks
    __shared__ __align__(8) uint64_t s_full[kStages];   // the loads of a stage have landed (and its slot is published)
    __shared__ __align__(8) uint64_t s_done[kStages];   // all computing warps are through with a stage
    __shared__ int s_abort;
    static_assert(kStages * S::kBytes + sizeof(s_group) + sizeof(s_slot) + sizeof(s_key) + 2 * sizeof(s_full) + 64 <= 227 * 1024,
                  "shared memory");

    ElxCtl* const ctl = a.ctl;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool skip = ctl->skip != 0;
    const int step = ctl->step;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&s_full[s], 1);
            mbar_init(&s_done[s], kWarps);
        }
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();

    const int64_t tile_lo = a.descs[a.first].tile_begin;
    const int64_t my_tiles = blockIdx.x < a.n_tiles ? (a.n_tiles - blockIdx.x + gridDim.x - 1) / gridDim.x : 0;

    if (warp == kWarps) {
        // The mover: lane 0 issues the copies.  What a tile is (its descriptor, segment, kind and dither keys) is worked out
        // for 16 tiles at a time, a tile per lane: done tile by tile it held the copies up, a tile being due every 1.4 us.
        // The slots of the batch before stay in use meanwhile, so there are two batches of them.
        Cursor8 cur;
        auto look_up = [&](int64_t k) {
            if (lane < kBatch && k + lane < my_tiles) {
                Slot8 slot;
                classify<DT>(a, tile_lo + blockIdx.x + (k + lane) * gridDim.x, skip, cur, slot);
                s_slot[(k + lane) % (2 * kBatch)] = slot;
            }
            __syncwarp();
            if (!skip) {
                for (int i = lane; i < kBatch * kWarps; i += 32) {
                    const int at = static_cast<int>((k + i / kWarps) % (2 * kBatch));
                    s_key[at][i % kWarps] = dither_key(step, s_slot[at].chunk, s_slot[at].e0 / kMomentBlock + i % kWarps);
                }
            }
            __syncwarp();
        };
        auto produce = [&](int64_t k, int s) {
            if (k % kBatch == 0) look_up(k);
            if (lane != 0) return;
            unsigned char* const at = s_dyn + s * S::kBytes;
            const Slot8& slot = s_slot[k % (2 * kBatch)];
            if (slot.kind == kWhole || slot.kind == kMixed) {
                const int64_t block = slot.e0 / kMomentBlock;
                mbar_arrive_expect_tx(&s_full[s], S::kLoaded);
                bulk_g2s(at + S::kP, slot.master + slot.e0, 4 * kTile, &s_full[s]);
                bulk_g2s(at + S::kG, static_cast<const T*>(slot.gsrc) + slot.e0, S::kGBytes, &s_full[s]);
                bulk_g2s(at + S::kM, slot.state_m + slot.e0, kTile, &s_full[s]);
                bulk_g2s(at + S::kV, slot.state_v + slot.e0, kTile, &s_full[s]);
                bulk_g2s(at + S::kEm, slot.exps_m + block, kWarps, &s_full[s]);
                bulk_g2s(at + S::kEv, slot.exps_v + block, kWarps, &s_full[s]);
            } else if (slot.kind == kRefresh) {
                mbar_arrive_expect_tx(&s_full[s], 4 * kTile);
                bulk_g2s(at + S::kP, slot.master + slot.e0, 4 * kTile, &s_full[s]);
            } else {
                mbar_arrive(&s_full[s]);   // nothing to load: publishes the slot
            }
        };
        for (int k = 0; k < my_tiles && k < kStages - 1; ++k) produce(k, k);
        int64_t k = 0;
        int s = 0;
        uint32_t parity = 0;
        bool gave_up = false;
        for (; k < my_tiles; ++k) {
            bool handed_over = false;
            for (uint32_t i = 0; i < kTmaSpinLimit && !handed_over; ++i) {
                handed_over = mbar_try_wait(&s_done[s], parity);
                if (!handed_over && *reinterpret_cast<volatile int*>(&s_abort)) break;
            }
            gave_up = __any_sync(0xFFFFFFFFu, !handed_over);
            if (gave_up) {
                s_abort = 1;
                break;
            }
            if (lane == 0) {
                const Slot8& slot = s_slot[k % (2 * kBatch)];
                unsigned char* const at = s_dyn + s * S::kBytes;
                const bool moments = slot.kind == kWhole || slot.kind == kMixed;
                if (moments || slot.kind == kRefresh)
                    bulk_s2g(static_cast<T*>(slot.lowp) + slot.e0, at + S::kG, S::kGBytes);
                if (moments) {
                    const int64_t block = slot.e0 / kMomentBlock;
                    bulk_s2g(slot.master + slot.e0, at + S::kP, 4 * kTile);
                    bulk_s2g(slot.state_m + slot.e0, at + S::kM, kTile);
                    bulk_s2g(slot.state_v + slot.e0, at + S::kV, kTile);
                    bulk_s2g(slot.exps_m + block, at + S::kEm, kWarps);
                    bulk_s2g(slot.exps_v + block, at + S::kEv, kWarps);
                }
                bulk_commit();
            }
            const int before = s == 0 ? kStages - 1 : s - 1;
            if (k + kStages - 1 < my_tiles) {
                if (lane == 0) bulk_wait_read<1>();   // the stage of tile k-1 has been read out by its stores
                produce(k + kStages - 1, before);
            }
            if (++s == kStages) {
                s = 0;
                parity ^= 1u;
            }
        }
        if (lane == 0) {
            if (gave_up) {
                // the loads already issued still target this CTA's shared memory: wait (bounded again) for them
                for (int64_t j = k; j < my_tiles && j < k + kStages - 1; ++j)
                    (void)mbar_wait_bounded(&s_full[j % kStages], static_cast<uint32_t>((j / kStages) & 1));
                atomicOr(&ctl->status, ELX_STAT_TIMEOUT);
            }
            bulk_wait_all();
        }
        return;
    }

    // the computing warps; the group constants take shape while the first tiles are on their way
    const float div = ctl->div_scale, inv_div = ctl->inv_div;
    const int div_mode = div > 0.0f ? (inv_div != 0.0f ? kMulInv : kTrueDiv) : kNoDiv;
    if (!skip && threadIdx.x < 2 * a.n_groups) derive_half(a.hyper[threadIdx.x >> 1], step, threadIdx.x & 1, s_group[threadIdx.x >> 1]);
    asm volatile("bar.sync 1, %0;" ::"n"(kComputing) : "memory");

    float nan_acc = 0.0f;
    bool bad_desc = false;
    Group8 k8 = {};
    int have = -1;
    bool l2 = false;
    int s = 0;
    uint32_t parity = 0;
    for (int64_t k = 0; k < my_tiles; ++k) {
        if (!mbar_wait_bounded(&s_full[s], parity)) {
            s_abort = 1;
            break;
        }
        const int slot_at = static_cast<int>(k) & (2 * kBatch - 1);
        const Slot8& slot = s_slot[slot_at];
        unsigned char* const at = s_dyn + s * S::kBytes;
        float* const sp = reinterpret_cast<float*>(at + S::kP) + warp * kMomentBlock;
        T* const sg = reinterpret_cast<T*>(at + S::kG) + warp * kMomentBlock;
        uint8_t *const scm = at + S::kM + warp * kMomentBlock, *const scv = at + S::kV + warp * kMomentBlock;

        int kind = slot.kind, group = slot.group, seg_lo = 0, seg_hi = -1;
        if (kind == kMixed && !block_segments(slot.segs, slot.n_segs, slot.seg, a.n_groups, slot.e0 + warp * kMomentBlock,
                                              slot.e0 + (warp + 1) * kMomentBlock, seg_lo, seg_hi, group))
            kind = kRefresh;   // this block of it
        if (kind == kWhole || kind == kMixed) {
            if (group >= 0 && group != have) {
                have = group;
                k8 = s_group[have];
                l2 = k8.wd_l2 != 0.0f;
            }
            const uint32_t key = s_key[slot_at][warp];
            const uint32_t em0 = at[S::kEm + warp], ev0 = at[S::kEv + warp];
            // a lane owns 2 x 4 consecutive elements, 128 apart: conflict-free accesses of whole words
            float2 p[4], m[4], v[4];
            const float dm = em0 ? __uint_as_float((em0 + 112u) << 23) : 0.0f;   // 2^(E - 15)
            const float dv = ev0 ? __uint_as_float((ev0 + 96u) << 23) : 0.0f;    // 2^(E - 31)
            float top_m = 0.0f, top_v = 0.0f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int i = h * 128 + lane * 4;
                const float4 pp = *reinterpret_cast<const float4*>(sp + i);
                const uint32_t cm = *reinterpret_cast<const uint32_t*>(scm + i), cv = *reinterpret_cast<const uint32_t*>(scv + i);
                float2 g[2];
                if constexpr (DT == ELX_F32) {
                    const float4 gg = *reinterpret_cast<const float4*>(sg + i);
                    g[0] = make_float2(gg.x, gg.y);
                    g[1] = make_float2(gg.z, gg.w);
                } else {
                    const uint2 gg = *reinterpret_cast<const uint2*>(sg + i);
                    g[0] = Lp<DT>::unpack2(gg.x);
                    g[1] = Lp<DT>::unpack2(gg.y);
                }
                p[2 * h] = make_float2(pp.x, pp.y);
                p[2 * h + 1] = make_float2(pp.z, pp.w);
                if (div_mode == kMulInv) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) g[j] = mul2(g[j], both(inv_div));
                } else if (div_mode == kTrueDiv) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) g[j] = make_float2(div_or_zero(g[j].x, div), div_or_zero(g[j].y, div));
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int q = 2 * h + j;
                    // sign and magnitude from the two ends of the byte, moved down by 4 to where fp32 has them
                    const int32_t m0 = static_cast<int32_t>(byte_to_top(cm, 2 * j)), m1 = static_cast<int32_t>(byte_to_top(cm, 2 * j + 1));
                    m[q] = mul2(make_float2(__int_as_float((m0 >> 4) & 0x87F00000), __int_as_float((m1 >> 4) & 0x87F00000)), both(dm));
                    v[q] = mul2(make_float2(__uint_as_float(byte_to_top(cv, 2 * j) >> 4),
                                                  __uint_as_float(byte_to_top(cv, 2 * j + 1) >> 4)), both(dv));
                    new_moments2(p[q], m[q], v[q], g[j], k8, l2);
                    top_m = max_nan(top_m, fabsf(m[q].x), fabsf(m[q].y));
                    top_v = max_nan(top_v, v[q].x, v[q].y);
                }
            }
            const uint32_t em = block_exponent(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(top_m)));
            const uint32_t ev = block_exponent(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(top_v)));
            if (group >= 0 && max(em, em0) <= kEasyM && max(ev, ev0) <= kEasyV) {
                const float xm = __uint_as_float((142u - em) << 23);   // 2^(15 - E)
                const float xv = __uint_as_float((158u - ev) << 23);   // 2^(31 - E)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int i = h * 128 + lane * 4;
                    uint32_t tm[4], tv[4];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int q = 2 * h + j;
                        const float2 zm = mul2(m[q], both(xm)), zv = mul2(v[q], both(xv));
                        const uint32_t r0 = dither_bits(key, i + 2 * j), r1 = dither_bits(key, i + 2 * j + 1);
                        // a shift by 4 drops the sign and lets the kept bits of a code end at bit 24: the code is the top byte
                        tm[2 * j] = ((__float_as_uint(zm.x) << 4) + __byte_perm(r0, 0, 0x4104)) | (__float_as_uint(zm.x) & 0x80000000u);
                        tm[2 * j + 1] = ((__float_as_uint(zm.y) << 4) + __byte_perm(r1, 0, 0x4104)) | (__float_as_uint(zm.y) & 0x80000000u);
                        tv[2 * j] = (__float_as_uint(zv.x) << 4) + __byte_perm(r0, 0, 0x4324);
                        tv[2 * j + 1] = (__float_as_uint(zv.y) << 4) + __byte_perm(r1, 0, 0x4324);
                        p[q] = new_param2(p[q], m[q], v[q], k8);
                    }
                    if (min(min(tv[0], tv[1]), min(tv[2], tv[3])) < 0x1000000u) {   // a code 0 stays only for a moment of 0
                        if (v[2 * h].x > 0.0f) tv[0] = max(tv[0], 0x1000000u);
                        if (v[2 * h].y > 0.0f) tv[1] = max(tv[1], 0x1000000u);
                        if (v[2 * h + 1].x > 0.0f) tv[2] = max(tv[2], 0x1000000u);
                        if (v[2 * h + 1].y > 0.0f) tv[3] = max(tv[3], 0x1000000u);
                    }
                    *reinterpret_cast<uint32_t*>(scm + i) = top_bytes(tm[0], tm[1], tm[2], tm[3]);
                    *reinterpret_cast<uint32_t*>(scv + i) = top_bytes(tv[0], tv[1], tv[2], tv[3]);
                    *reinterpret_cast<float4*>(sp + i) = make_float4(p[2 * h].x, p[2 * h].y, p[2 * h + 1].x, p[2 * h + 1].y);
                    if constexpr (DT == ELX_F32) {
                        *reinterpret_cast<float4*>(sg + i) = make_float4(p[2 * h].x, p[2 * h].y, p[2 * h + 1].x, p[2 * h + 1].y);
                    } else {
                        *reinterpret_cast<uint2*>(sg + i) = make_uint2(Lp<DT>::pack2(p[2 * h].x, p[2 * h].y),
                                                                       Lp<DT>::pack2(p[2 * h + 1].x, p[2 * h + 1].y));
                    }
                }
                __syncwarp();   // every lane has read the old exponents
                if (lane == 0) {
                    at[S::kEm + warp] = static_cast<uint8_t>(em);
                    at[S::kEv + warp] = static_cast<uint8_t>(ev);
                }
            } else {
                const BlockAt b = {sp, sg, sg, scm, scv, at + S::kEm + warp, at + S::kEv + warp, slot.e0 + warp * kMomentBlock,
                                   kMomentBlock, slot.segs, seg_lo, seg_hi, group};
                update_block<DT>(b, s_group, a.n_groups, key, div_mode, div, inv_div, nan_acc);
            }
            fence_async_smem();   // the bulk stores read what the threads just wrote
        } else if (kind == kRefresh) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int i = h * 128 + lane * 4;
                const float4 pp = *reinterpret_cast<const float4*>(sp + i);
                if constexpr (DT == ELX_F32) *reinterpret_cast<float4*>(sg + i) = pp;
                else *reinterpret_cast<uint2*>(sg + i) = make_uint2(Lp<DT>::pack2(pp.x, pp.y), Lp<DT>::pack2(pp.z, pp.w));
            }
            fence_async_smem();
        } else if (kind == kRagged) {
            const int64_t b0 = slot.e0 + warp * kMomentBlock, b1 = min(b0 + kMomentBlock, slot.e1);
            T* const lowp = static_cast<T*>(slot.lowp);
            if (b0 < b1) {
                if (!skip && (group >= 0 || block_segments(slot.segs, slot.n_segs, slot.seg, a.n_groups, b0, b1, seg_lo, seg_hi, group))) {
                    const int64_t block = b0 / kMomentBlock;
                    const BlockAt b = {slot.master + b0, static_cast<const T*>(slot.gsrc) + b0, lowp + b0, slot.state_m + b0,
                                       slot.state_v + b0, slot.exps_m + block, slot.exps_v + block, b0, static_cast<int>(b1 - b0),
                                       slot.segs, seg_lo, seg_hi, group};
                    update_block<DT>(b, s_group, a.n_groups, s_key[slot_at][warp], div_mode, div, inv_div, nan_acc);
                } else {
                    for (int64_t e = b0 + lane; e < b1; e += 32) lowp[e] = Lp<DT>::from_float(slot.master[e]);
                }
            }
        } else {
            bad_desc = true;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_done[s]);
        if (++s == kStages) {
            s = 0;
            parity ^= 1u;
        }
    }

    const unsigned late = __ballot_sync(0xFFFFFFFFu, nan_acc != nan_acc);
    if (lane == 0) {
        if (late) {
            atomicOr(&ctl->late_inf, 1u);
            atomicOr(&ctl->status, ELX_STAT_LATE_INF);
        }
        if (bad_desc) atomicOr(&ctl->status, ELX_STAT_BAD_DESC);
    }
}

template <int DT>
int launch_adam8(const Adam8Args& a, cudaStream_t s) {
    constexpr int smem = Stage8<DT>::kStages * Stage8<DT>::kBytes;
    // the opt-in to more than 48 KB of dynamic shared memory is per device: once for each ordinal
    static bool opted_in[64];
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
        (void)cudaGetLastError();
        return ELX_ERR_NODEVICE;
    }
    if (!opted_in[dev]) {
        const cudaError_t attr = cudaFuncSetAttribute(adam8_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (attr != cudaSuccess) {
            const int rc = record_cuda(attr);
            (void)cudaGetLastError();
            return rc;
        }
        opted_in[dev] = true;
    }
    const int grid = grid_for(a.n_tiles, 1);
    if (grid < 0) return grid;
    adam8_kernel<DT><<<grid, kThreads, smem, s>>>(a);
    return record_cuda(cudaGetLastError());
}

// ------------------------------------------------------------------------------------------------
// conversion
// ------------------------------------------------------------------------------------------------

constexpr int kConvThreads = 256;
constexpr int kPair = 2 * kMomentBlock;   // elements a warp converts at a time: 16 lanes per block, 16 elements per lane

// One block by one warp, element by element: the end of a shard, and arrays that are not aligned.
template <class M>
__device__ __noinline__ void pack_block(const float* __restrict__ x, uint8_t* state, int64_t n, int64_t block) {
    const int lane = threadIdx.x & 31;
    const int64_t b0 = block * kMomentBlock;
    if (b0 >= n) return;
    float f[8];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int64_t e = b0 + lane + 32 * j;
        f[j] = e < n ? x[e] : 0.0f;
        top = max(top, __float_as_uint(f[j]) & 0x7FFFFFFFu);
    }
    const uint32_t exp = block_exponent(__reduce_max_sync(0xFFFFFFFFu, top));
    const float scale = encode_scale(exp);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int64_t e = b0 + lane + 32 * j;
        if (e < n) state[e] = static_cast<uint8_t>(encode<M>(f[j], scale, kRoundNearest));
    }
    if (lane == 0) state[moment_exps_at(n) + block] = static_cast<uint8_t>(exp);
}

template <class M>
__device__ __forceinline__ void pack_pair(const float* __restrict__ x, uint8_t* state, int64_t n, int64_t pair) {
    const int lane = threadIdx.x & 31;
    const int64_t e = pair * kPair + lane * 16;
    float f[16];
    uint32_t top = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const U8 r = ld256(x + e + 8 * h);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            f[8 * h + j] = __uint_as_float(r.x[j]);
            top = max(top, r.x[j] & 0x7FFFFFFFu);
        }
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    const uint32_t exp = block_exponent(top);
    const float scale = encode_scale(exp);
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 16; ++j) w[j / 4] |= encode<M>(f[j], scale, kRoundNearest) << (8 * (j & 3));
    *reinterpret_cast<uint4*>(state + e) = make_uint4(w[0], w[1], w[2], w[3]);
    if ((lane & 15) == 0) state[moment_exps_at(n) + pair * 2 + (lane >> 4)] = static_cast<uint8_t>(exp);
}

// Bound by the bytes: 8 in and 2 out per element; 64 Mi elements in 106 us (6.4 TB/s).  Back into fp32: 110 us (6.1 TB/s),
// into bf16 70 us (5.8 TB/s; that form spills 20 bytes per thread).
__global__ void __launch_bounds__(kConvThreads) pack_kernel(const float* __restrict__ m, const float* __restrict__ v, int64_t n,
                                                            uint8_t* state_m, uint8_t* state_v, int vec) {
    const int64_t pairs = (n + kPair - 1) / kPair, stride = static_cast<int64_t>(gridDim.x) * (kConvThreads / 32);
    for (int64_t q = blockIdx.x * (kConvThreads / 32) + (threadIdx.x >> 5); q < pairs; q += stride) {
        if (vec && (q + 1) * kPair <= n) {
            pack_pair<FirstMoment>(m, state_m, n, q);
            pack_pair<SecondMoment>(v, state_v, n, q);
        } else {
            for (int64_t b = 2 * q; b < 2 * q + 2; ++b) {
                pack_block<FirstMoment>(m, state_m, n, b);
                pack_block<SecondMoment>(v, state_v, n, b);
            }
        }
    }
    if (blockIdx.x == 0 && threadIdx.x < 32) {   // the padding: fewer than 16 bytes behind the codes and behind the exponents
        const int64_t exps = moment_exps_at(n), end = exps + (n + kMomentBlock - 1) / kMomentBlock;
        const int64_t at = threadIdx.x < 16 ? n + threadIdx.x : end + threadIdx.x - 16;
        if (at < (threadIdx.x < 16 ? exps : moment_state_bytes(n))) state_m[at] = state_v[at] = 0;
    }
}

template <class M, int DT>
__device__ __forceinline__ void unpack_codes(const uint4& c, float scale, typename Lp<DT>::T* out) {
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
    float f[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) f[j] = decode<M>((w[j / 4] >> (8 * (j & 3))) & 0xFFu, scale);
    if constexpr (DT == ELX_F32) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            U8 r;
#pragma unroll
            for (int j = 0; j < 8; ++j) r.x[j] = __float_as_uint(f[8 * h + j]);
            st256(out + 8 * h, r);
        }
    } else {
        U8 r;
#pragma unroll
        for (int j = 0; j < 8; ++j) r.x[j] = Lp<DT>::pack2(f[2 * j], f[2 * j + 1]);
        st256(out, r);
    }
}

template <int DT>
__global__ void __launch_bounds__(kConvThreads, 4) unpack_kernel(const uint8_t* __restrict__ state_m, const uint8_t* __restrict__ state_v,
                                                              int64_t n, void* m, void* v, int vec) {
    using T = typename Lp<DT>::T;
    T *const om = static_cast<T*>(m), *const ov = static_cast<T*>(v);
    const uint8_t *const exps_m = state_m + moment_exps_at(n), *const exps_v = state_v + moment_exps_at(n);
    const int lane = threadIdx.x & 31;
    const int64_t pairs = (n + kPair - 1) / kPair, stride = static_cast<int64_t>(gridDim.x) * (kConvThreads / 32);
    for (int64_t q = blockIdx.x * (kConvThreads / 32) + (threadIdx.x >> 5); q < pairs; q += stride) {
        const int64_t e = q * kPair + lane * 16;
        if (vec && (q + 1) * kPair <= n) {
            const uint4 cm = __ldcs(reinterpret_cast<const uint4*>(state_m + e)), cv = __ldcs(reinterpret_cast<const uint4*>(state_v + e));
            const float sm = decode_scale(exps_m[2 * q + (lane >> 4)]), sv = decode_scale(exps_v[2 * q + (lane >> 4)]);
            unpack_codes<FirstMoment, DT>(cm, sm, om + e);
            unpack_codes<SecondMoment, DT>(cv, sv, ov + e);
        } else {
            // element by element: the codes of one moment after the other, all on their way before the first is decoded
            const int64_t first = q * kPair + lane;
            const uint8_t* const codes[2] = {state_m, state_v};
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                uint32_t c[16];
                float scale[2];
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    scale[j] = q * kPair + j * kMomentBlock < n ? decode_scale((k ? exps_v : exps_m)[2 * q + j]) : 0.0f;
#pragma unroll
                for (int j = 0; j < 16; ++j) c[j] = first + 32 * j < n ? codes[k][first + 32 * j] : 0u;
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (first + 32 * j < n)
                        (k ? ov : om)[first + 32 * j] = Lp<DT>::from_float(k ? decode<SecondMoment>(c[j], scale[j / 8])
                                                                              : decode<FirstMoment>(c[j], scale[j / 8]));
            }
        }
    }
}

// Blocks per SM, of which four run at a time: packing runs best in many turns of short blocks, unpacking, which writes more than
// it reads, in two (64 Mi elements: packing 105.7 us with 64, 110.5 us with 8; unpacking into bf16 70.9 us and 69.8 us).
int conversion_grid(int64_t n, int per_sm) {
    const int64_t per_block = static_cast<int64_t>(kConvThreads / 32) * kPair;
    return grid_for((n + per_block - 1) / per_block, per_sm);
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
    const int vec = aligned(exp_avg, 32) && aligned(exp_avg_sq, 32) && aligned(state_m, 16) && aligned(state_v, 16);
    const int grid = conversion_grid(n, 64);
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
    const int vec = aligned(exp_avg, 32) && aligned(exp_avg_sq, 32) && aligned(state_m, 16) && aligned(state_v, 16);
    const int grid = conversion_grid(n, 8);
    if (grid < 0) return grid;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const uint8_t *sm = static_cast<const uint8_t*>(state_m), *sv = static_cast<const uint8_t*>(state_v);
    if (dtype == ELX_F32) unpack_kernel<ELX_F32><<<grid, kConvThreads, 0, s>>>(sm, sv, n, exp_avg, exp_avg_sq, vec);
    else unpack_kernel<ELX_BF16><<<grid, kConvThreads, 0, s>>>(sm, sv, n, exp_avg, exp_avg_sq, vec);
    return record_cuda(cudaGetLastError());
}

}  // extern "C"
