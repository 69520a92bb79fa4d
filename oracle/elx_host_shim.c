/*
 * TEST INFRASTRUCTURE — the elx_* C ABI implemented on HOST memory with the CPU oracle.
 *
 * The test-suite loads this in place of libelixir_b200.so (tests/_dist_workers.py) to run the host-side
 * logic of the package — chunk geometry, collectives over gloo, the ElixirOptimizer state machine —
 * on machines without a GPU.  The product never loads it.  Pointers are host pointers, the stream
 * argument is ignored, every call completes before it returns.  Arithmetic: elx_oracle.c (double
 * precision evaluation of the update, rounded to fp32).
 */
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "elixir_b200.h"

int orc_probe(const void* g, int dtype, int64_t n_valid);
double orc_l2sq(const void* g, int dtype, int64_t n_valid);
void orc_cast(const float* src, void* dst, int dtype, int64_t n);
void orc_ctl_init(ElxCtl* ctl, float initial_scale);
void orc_step_begin(ElxCtl* ctl, ElxScalerCfg cfg, const float* norm_sq);
void orc_adam_f64(float* p, float* m, float* v, const void* g, int dtype, int64_t begin, int64_t end, ElxHyper h,
                  int step, float div_scale);

static int dtype_ok(int dt) { return dt == ELX_F16 || dt == ELX_BF16 || dt == ELX_F32; }
static int dtype_bytes(int dt) { return dt == ELX_F32 ? 4 : 2; }

int elx_version(void) { return ELX_ABI_VERSION; }
const char* elx_strerror(int status) { return status == ELX_OK ? "ok" : "host shim: argument rejected"; }
const char* elx_last_cuda_error(void) { return ""; }
int elx_set_tuning(const char* name, int value) {
    (void)value;
    return name ? ELX_OK : ELX_ERR_NULL;
}
int64_t elx_probe_scratch_elems(int64_t n_tiles) { return n_tiles < 0 ? 0 : n_tiles; }
int64_t elx_grad_check_static_max_elems(void) { return (int64_t)16384 * ELX_TILE; }

int elx_ctl_init(ElxCtl* ctl, float initial_scale, void* stream) {
    (void)stream;
    if (!ctl) return ELX_ERR_NULL;
    orc_ctl_init(ctl, initial_scale);
    return ELX_OK;
}

int elx_step_begin(ElxCtl* ctl, ElxScalerCfg cfg, const float* norm_sq, uint32_t* chunk_flags, int n_chunk_flags,
                   void* stream) {
    (void)stream;
    if (!ctl) return ELX_ERR_NULL;
    if (cfg.max_norm > 0.0f && !norm_sq) return ELX_ERR_NULL;
    if (n_chunk_flags < 0) return ELX_ERR_SIZE;
    if (ctl->status & ELX_STAT_TIMEOUT) {
        /* a wait gave up earlier: skip without touching the loss scaler (no reference counterpart) */
        ctl->skip = 1;
        ctl->skipped_steps += 1;
        ctl->forced_skips += 1;
        ctl->div_scale = -1.0f;
        ctl->inv_div = 0.0f;
        ctl->found_inf = 0;
    } else {
        orc_step_begin(ctl, cfg, norm_sq);
    }
    for (int i = 0; chunk_flags && i < n_chunk_flags; ++i) chunk_flags[i] = 0;
    return ELX_OK;
}

static const void* grad_of(const ElxChunkDesc* d) { return d->grad_src ? d->grad_src : d->grad_param; }

static int probe_common(const void* g, int dtype, int64_t n_valid, uint32_t* flag, ElxCtl* ctl, float* l2sq) {
    if (!g) return ELX_ERR_NULL;
    if (!dtype_ok(dtype)) return ELX_ERR_DTYPE;
    if (n_valid < 0) return ELX_ERR_SIZE;
    if (orc_probe(g, dtype, n_valid)) {
        if (flag) *flag = 1;
        if (ctl) ctl->found_inf = 1;
    }
    if (l2sq) *l2sq = (float)orc_l2sq(g, dtype, n_valid);
    return ELX_OK;
}

int elx_grad_check(const void* g, int dtype, int64_t n_valid, uint32_t* flag, ElxCtl* ctl, float* l2sq, float* scratch,
                   int64_t scratch_elems, void* stream) {
    (void)scratch;
    (void)scratch_elems;
    (void)stream;
    return probe_common(g, dtype, n_valid, flag, ctl, l2sq);
}

int elx_grad_check_static(const void* g, int dtype, int64_t n_valid, uint32_t* flag, ElxCtl* ctl, float* l2sq,
                          void* stream) {
    (void)stream;
    if (l2sq && g && dtype_ok(dtype) && n_valid > elx_grad_check_static_max_elems()) return ELX_ERR_CAPACITY;
    return probe_common(g, dtype, n_valid, flag, ctl, l2sq);
}

int elx_reduce_epilogue(const void* src, void* dst, int dtype, int64_t n_shard, int64_t n_valid, uint32_t* flag,
                        ElxCtl* ctl, float* l2sq, float* scratch, int64_t scratch_elems, void* stream) {
    (void)scratch;
    (void)scratch_elems;
    (void)stream;
    if (!src || !dst) return ELX_ERR_NULL;
    if (!dtype_ok(dtype)) return ELX_ERR_DTYPE;
    if (n_shard < 0 || n_valid < 0 || n_valid > n_shard) return ELX_ERR_SIZE;
    memmove(dst, src, (size_t)n_shard * dtype_bytes(dtype));
    return probe_common(src, dtype, n_valid, flag, ctl, l2sq);
}

float orc_f16_to_f32(uint16_t h);
float orc_bf16_to_f32(uint16_t h);

int elx_widen(const void* src, int dtype, float* dst, int64_t n, void* stream) {
    (void)stream;
    if (!src || !dst) return ELX_ERR_NULL;
    if (dtype != ELX_F16 && dtype != ELX_BF16) return ELX_ERR_DTYPE;
    if (n < 0) return ELX_ERR_SIZE;
    const uint16_t* in = (const uint16_t*)src;
    for (int64_t i = 0; i < n; ++i) dst[i] = dtype == ELX_F16 ? orc_f16_to_f32(in[i]) : orc_bf16_to_f32(in[i]);
    return ELX_OK;
}

int elx_narrow_epilogue(const float* src, void* dst, int dtype, int64_t n_shard, int64_t n_valid, uint32_t* flag,
                        ElxCtl* ctl, void* stream) {
    (void)stream;
    if (!src || !dst) return ELX_ERR_NULL;
    if (dtype != ELX_F16 && dtype != ELX_BF16) return ELX_ERR_DTYPE;
    if (n_shard < 0 || n_valid < 0 || n_valid > n_shard) return ELX_ERR_SIZE;
    orc_cast(src, dst, dtype, n_shard);
    return probe_common(dst, dtype, n_valid, flag, ctl, 0);
}

int elx_grad_check_multi(const ElxChunkDesc* descs, int first, int count, int64_t n_tiles, int dtype,
                         uint32_t* chunk_flags, ElxCtl* ctl, float* chunk_l2sq, float* total_l2sq, float* scratch,
                         int64_t scratch_elems, void* stream) {
    (void)n_tiles;
    (void)scratch;
    (void)scratch_elems;
    (void)stream;
    if (!descs) return ELX_ERR_NULL;
    double total = 0.0;
    for (int c = first; c < first + count; ++c) {
        if (descs[c].dtype != dtype) {
            if (ctl) ctl->status |= ELX_STAT_BAD_DESC;
            continue;
        }
        float l2 = 0.0f;
        int rc = probe_common(grad_of(&descs[c]), dtype, descs[c].n_valid, chunk_flags ? &chunk_flags[c] : 0, ctl,
                              (chunk_l2sq || total_l2sq) ? &l2 : 0);
        if (rc != ELX_OK) return rc;
        if (chunk_l2sq) chunk_l2sq[c] = l2;
        total += l2;
    }
    if (total_l2sq) *total_l2sq = (float)total;
    return ELX_OK;
}

static void step_one(const ElxChunkDesc* d, const ElxSeg* segs, const ElxHyper* hyper, int n_groups,
                     const ElxCtl* ctl) {
    if (!ctl->skip) {
        for (int s = d->seg_first; s < d->seg_first + d->seg_count; ++s) {
            if (segs[s].group < 0 || segs[s].group >= n_groups) continue;
            orc_adam_f64(d->master, d->exp_avg, d->exp_avg_sq, grad_of(d), d->dtype, segs[s].begin, segs[s].end,
                         hyper[segs[s].group], ctl->step, ctl->div_scale);
        }
    }
    orc_cast(d->master, d->grad_param, d->dtype, d->n_shard);
}

int elx_adam_multi(const ElxChunkDesc* descs, int first, int count, int64_t n_tiles, int dtype, const ElxSeg* segs,
                   const ElxHyper* hyper, int n_groups, ElxCtl* ctl, void* stream) {
    (void)n_tiles;
    (void)stream;
    if (!descs || !ctl) return ELX_ERR_NULL;
    if (n_groups > 64) return ELX_ERR_CAPACITY;
    for (int c = first; c < first + count; ++c) {
        if (descs[c].dtype != dtype) {
            ctl->status |= ELX_STAT_BAD_DESC;
            continue;
        }
        step_one(&descs[c], segs, hyper, n_groups, ctl);
    }
    return ELX_OK;
}

int elx_adam_chunk(float* master, float* exp_avg, float* exp_avg_sq, void* grad_param, int dtype, int64_t n_valid,
                   int64_t n_shard, ElxHyper hyper, ElxCtl* ctl, void* stream) {
    (void)stream;
    if (!master || !exp_avg || !exp_avg_sq || !grad_param || !ctl) return ELX_ERR_NULL;
    if (n_valid < 0 || n_valid > n_shard) return ELX_ERR_SIZE;
    ElxChunkDesc d;
    memset(&d, 0, sizeof(d));
    d.master = master;
    d.exp_avg = exp_avg;
    d.exp_avg_sq = exp_avg_sq;
    d.grad_param = grad_param;
    d.n_shard = n_shard;
    d.n_valid = n_valid;
    d.seg_count = n_valid > 0 ? 1 : 0;
    d.dtype = dtype;
    ElxSeg seg = {0, n_valid, 0, 0};
    step_one(&d, &seg, &hyper, 1, ctl);
    return ELX_OK;
}

int elx_cast_copyback(const float* master, void* dst, int dtype, int64_t n, void* stream) {
    (void)stream;
    if (!master || !dst) return ELX_ERR_NULL;
    if (!dtype_ok(dtype)) return ELX_ERR_DTYPE;
    orc_cast(master, dst, dtype, n);
    return ELX_OK;
}

/* The NVLink entry points have no host-memory form: they need peer-mapped device memory. */
int elx_enable_peer_access(int peer_device) {
    (void)peer_device;
    return ELX_ERR_NODEVICE;
}
int elx_peer_barrier(ElxPeerTable flags, uint32_t epoch, ElxCtl* ctl, int exchange_overflow, int timeout_ms,
                     void* stream) {
    (void)flags; (void)epoch; (void)ctl; (void)exchange_overflow; (void)timeout_ms; (void)stream;
    return ELX_ERR_NODEVICE;
}
int elx_pull_reduce_multi(const ElxChunkDesc* descs, int first, int count, int64_t n_tiles, int dtype,
                          ElxPeerTable grads, const int64_t* block_off, const int64_t* stage_off,
                          uint32_t* chunk_flags, ElxCtl* ctl, void* stream) {
    (void)descs; (void)first; (void)count; (void)n_tiles; (void)dtype; (void)grads; (void)block_off; (void)stage_off;
    (void)chunk_flags; (void)ctl; (void)stream;
    return ELX_ERR_NODEVICE;
}
int elx_adam_multi_shadow(const ElxChunkDesc* descs, const ElxChunkDesc* shadow, int first, int count,
                          int64_t n_tiles, int dtype, const ElxSeg* segs, const ElxHyper* hyper, int n_groups,
                          ElxCtl* ctl, void* stream) {
    (void)n_tiles;
    (void)stream;
    if (!descs || !shadow || !ctl) return ELX_ERR_NULL;
    if (n_groups > 64) return ELX_ERR_CAPACITY;
    for (int c = first; c < first + count; ++c) {
        const ElxChunkDesc* d = &descs[c];
        const ElxChunkDesc* o = &shadow[c];
        if (d->dtype != dtype || o->n_shard != d->n_shard) {
            ctl->status |= ELX_STAT_BAD_DESC;
            continue;
        }
        if (ctl->skip) {
            orc_cast(d->master, d->grad_param, d->dtype, d->n_shard);
            continue;
        }
        for (int s = d->seg_first; s < d->seg_first + d->seg_count; ++s) {
            if (segs[s].group < 0 || segs[s].group >= n_groups) continue;
            const int64_t b = segs[s].begin, n = segs[s].end - segs[s].begin;
            memcpy(o->master + b, d->master + b, (size_t)n * sizeof(float));
            memcpy(o->exp_avg + b, d->exp_avg + b, (size_t)n * sizeof(float));
            memcpy(o->exp_avg_sq + b, d->exp_avg_sq + b, (size_t)n * sizeof(float));
            orc_adam_f64(o->master, o->exp_avg, o->exp_avg_sq, grad_of(d), d->dtype, segs[s].begin, segs[s].end,
                         hyper[segs[s].group], ctl->step, ctl->div_scale);
        }
        orc_cast(o->master, d->grad_param, d->dtype, d->n_shard);
    }
    return ELX_OK;
}

/* ---- single-pass step over two sets of state (one rank; the collective form needs NVLink) ---- */

static void forced_skip(ElxCtl* ctl) {
    ctl->skip = 1;
    ctl->skipped_steps += 1;
    ctl->forced_skips += 1;
    ctl->div_scale = -1.0f;
    ctl->inv_div = 0.0f;
    ctl->found_inf = 0;
}

int elx_step_begin_optimistic(ElxCtl* ctl, ElxScalerCfg cfg, uint32_t* chunk_flags, int n_chunk_flags, void* stream) {
    (void)stream;
    if (!ctl) return ELX_ERR_NULL;
    if (cfg.max_norm > 0.0f) return ELX_ERR_ARG;
    ctl->repair = 0;
    if (ctl->status & ELX_STAT_TIMEOUT) {
        forced_skip(ctl);
        ctl->spec_state = 2;
    } else if (ctl->found_inf) {
        orc_step_begin(ctl, cfg, 0);
        ctl->spec_state = 2;
    } else {
        ctl->saved_scale = ctl->scale;
        ctl->saved_growth_step = ctl->growth_step;
        ctl->saved_hysteresis_step = ctl->hysteresis_step;
        ctl->saved_step = ctl->step;
        orc_step_begin(ctl, cfg, 0);
        ctl->spec_state = 1;
    }
    for (int i = 0; chunk_flags && i < n_chunk_flags; ++i) chunk_flags[i] = 0;
    return ELX_OK;
}

int elx_step_commit(ElxCtl* ctl, ElxScalerCfg cfg, uint32_t* chunk_flags, int n_chunk_flags, void* stream) {
    (void)stream;
    if (!ctl) return ELX_ERR_NULL;
    if (ctl->spec_state == 1) {
        const int expired = (ctl->status & ELX_STAT_TIMEOUT) != 0;
        if (expired || ctl->found_inf) {
            ctl->scale = ctl->saved_scale;
            ctl->growth_step = ctl->saved_growth_step;
            ctl->hysteresis_step = ctl->saved_hysteresis_step;
            ctl->step = ctl->saved_step;
            if (expired) {
                forced_skip(ctl);
            } else {
                ctl->found_inf = 1;
                orc_step_begin(ctl, cfg, 0);
            }
            ctl->repair = 1;
        } else {
            ctl->cur_set ^= 1u;
        }
    }
    ctl->spec_state = 0;
    ctl->found_inf = 0;
    for (int i = 0; chunk_flags && i < n_chunk_flags; ++i) chunk_flags[i] = 0;
    return ELX_OK;
}

int elx_adam_multi_single_pass(const ElxChunkDesc* descs, const ElxChunkDesc* shadow, int first, int count,
                               int64_t n_tiles, int dtype, const ElxSeg* segs, const ElxHyper* hyper, int n_groups,
                               ElxCtl* ctl, uint32_t* chunk_flags, ElxPeerTable grads, ElxPeerTable gather,
                               const int64_t* block_off, const void* grads_mc, void* gather_mc, void* stream) {
    (void)n_tiles; (void)grads; (void)block_off; (void)stream;
    if (!descs || !shadow || !ctl) return ELX_ERR_NULL;
    if (gather.world > 0 || grads_mc || gather_mc) return ELX_ERR_NODEVICE;
    if (n_groups > 64) return ELX_ERR_CAPACITY;
    const ElxChunkDesc* src = ctl->cur_set ? shadow : descs;
    const ElxChunkDesc* dst = ctl->cur_set ? descs : shadow;
    for (int c = first; c < first + count; ++c) {
        const ElxChunkDesc* d = &src[c];
        const ElxChunkDesc* o = &dst[c];
        if (d->dtype != dtype || o->n_shard != d->n_shard) {
            ctl->status |= ELX_STAT_BAD_DESC;
            continue;
        }
        if (ctl->skip) {
            orc_cast(d->master, d->grad_param, d->dtype, d->n_shard);
            continue;
        }
        if (orc_probe(grad_of(d), d->dtype, d->n_valid)) {
            ctl->found_inf = 1;
            if (chunk_flags) chunk_flags[c] = 1;
        }
        for (int s = d->seg_first; s < d->seg_first + d->seg_count; ++s) {
            if (segs[s].group < 0 || segs[s].group >= n_groups) continue;
            const int64_t b = segs[s].begin, n = segs[s].end - segs[s].begin;
            memcpy(o->master + b, d->master + b, (size_t)n * sizeof(float));
            memcpy(o->exp_avg + b, d->exp_avg + b, (size_t)n * sizeof(float));
            memcpy(o->exp_avg_sq + b, d->exp_avg_sq + b, (size_t)n * sizeof(float));
            orc_adam_f64(o->master, o->exp_avg, o->exp_avg_sq, grad_of(d), d->dtype, segs[s].begin, segs[s].end,
                         hyper[segs[s].group], ctl->step, ctl->div_scale);
        }
        orc_cast(o->master, d->grad_param, d->dtype, d->n_shard);
    }
    return ELX_OK;
}

int elx_adam_multi_repair(const ElxChunkDesc* descs, const ElxChunkDesc* shadow, int first, int count, int64_t n_tiles,
                          int dtype, ElxCtl* ctl, ElxPeerTable gather, const int64_t* block_off, void* gather_mc,
                          void* stream) {
    (void)n_tiles; (void)dtype; (void)block_off; (void)gather_mc; (void)stream;
    if (!descs || !shadow || !ctl) return ELX_ERR_NULL;
    if (gather.world > 0) return ELX_ERR_NODEVICE;
    if (!ctl->repair) return ELX_OK;
    const ElxChunkDesc* src = ctl->cur_set ? shadow : descs;
    for (int c = first; c < first + count; ++c) orc_cast(src[c].master, src[c].grad_param, src[c].dtype, src[c].n_shard);
    return ELX_OK;
}

int elx_adam_multi_hostmem(const ElxChunkDesc* descs, int first, int count, int64_t n_tiles, int dtype,
                           const ElxSeg* segs, const ElxHyper* hyper, int n_groups, ElxCtl* ctl, void* stream) {
    return elx_adam_multi(descs, first, count, n_tiles, dtype, segs, hyper, n_groups, ctl, stream);
}

int elx_adam_multi_push(const ElxChunkDesc* descs, int first, int count, int64_t n_tiles, int dtype,
                        const ElxSeg* segs, const ElxHyper* hyper, int n_groups, ElxCtl* ctl, ElxPeerTable gather,
                        const int64_t* block_off, void* stream) {
    (void)descs; (void)first; (void)count; (void)n_tiles; (void)dtype; (void)segs; (void)hyper; (void)n_groups;
    (void)ctl; (void)gather; (void)block_off; (void)stream;
    return ELX_ERR_NODEVICE;
}
int elx_adam_multi_pull_push(const ElxChunkDesc* descs, int first, int count, int64_t n_tiles, int dtype,
                             const ElxSeg* segs, const ElxHyper* hyper, int n_groups, ElxCtl* ctl, ElxPeerTable grads,
                             ElxPeerTable gather, const int64_t* block_off, void* stream) {
    (void)descs; (void)first; (void)count; (void)n_tiles; (void)dtype; (void)segs; (void)hyper; (void)n_groups;
    (void)ctl; (void)grads; (void)gather; (void)block_off; (void)stream;
    return ELX_ERR_NODEVICE;
}
int elx_multimem_reduce(const void* src_mc, void* dst, int dtype, int64_t n, void* stream) {
    (void)src_mc; (void)dst; (void)dtype; (void)n; (void)stream;
    return ELX_ERR_NODEVICE;
}
int elx_ipc_open(const void* handle, void** base) {
    (void)handle; (void)base;
    return ELX_ERR_NODEVICE;
}
int elx_ipc_close(void* base) {
    (void)base;
    return ELX_ERR_NODEVICE;
}
int elx_peek_u32(const void* device_ptr, uint32_t* value) {
    if (!device_ptr || !value) return ELX_ERR_NULL;
    *value = *(const uint32_t*)device_ptr;
    return ELX_OK;
}
int elx_peer_alloc(int64_t bytes, void** ptr, void* handle) {
    (void)bytes; (void)ptr; (void)handle;
    return ELX_ERR_NODEVICE;
}
int elx_peer_free(void* ptr) {
    (void)ptr;
    return ELX_ERR_NODEVICE;
}
int elx_copy_async(void* dst, const void* src, int64_t bytes, void* stream) {
    (void)stream;
    if (!dst || !src) return ELX_ERR_NULL;
    memmove(dst, src, (size_t)bytes);
    return ELX_OK;
}

/* ---- the update with both moments in 8 bits ---- */

static float bits_f32(uint32_t u) {
    float f;
    memcpy(&f, &u, 4);
    return f;
}
static uint32_t f32_bits(float f) {
    uint32_t u;
    memcpy(&u, &f, 4);
    return u;
}
static int64_t exps_at(int64_t n) { return (n + 15) / 16 * 16; }
static int64_t blocks_of(int64_t n) { return (n + ELX_MOMENT_BLOCK - 1) / ELX_MOMENT_BLOCK; }

int64_t elx_moment_state_bytes(int64_t n) { return n < 0 ? ELX_ERR_SIZE : exps_at(n) + (blocks_of(n) + 15) / 16 * 16; }

static double pow2(int e) { return ldexp(1.0, e); }

/* value of a code; `first`: the signed moment */
static float code_value(uint8_t c, uint8_t e, int first) {
    if (e == 255) return bits_f32(0x7FC00000u);
    if (e == 0) return 0.0f;
    const int bias = first ? 15 : 31, mag = first ? c & 127 : c, f = mag >> 3, t = mag & 7;
    const double v = f ? (1.0 + t / 8.0) * pow2(f - bias) : t / 8.0 * pow2(1 - bias);
    const float x = (float)(v * pow2((int)e - 127));
    return first && (c & 128) ? -x : x;
}

static uint8_t block_exp(const float* x, int n) {
    uint32_t top = 0;
    for (int i = 0; i < n; ++i) {
        const uint32_t u = f32_bits(x[i]) & 0x7FFFFFFFu;
        if (u > top) top = u;
    }
    if (top >= 0x7F800000u) return 255;
    if (top == 0) return 0;
    uint32_t e = (top + 0xFFFFFu) >> 23;
    return (uint8_t)(e < 1 ? 1 : e > 253 ? 253 : e);
}

/* `up` in [0, 1): how far towards the next code a value is pushed before the fraction is dropped (0.5: nearest) */
static uint8_t code_of(float x, uint8_t e, int first, double up) {
    const int bias = first ? 15 : 31, top = first ? 127 : 255, sign = first && (f32_bits(x) >> 31) ? 128 : 0;
    if (e == 0 || e == 255) return (uint8_t)sign;
    const double a = fabs((double)x) / pow2((int)e - 127);
    int f = bias;                                        /* exponent field of the binade that holds a (1: or below) */
    while (f > 1 && a < pow2(f - bias)) --f;
    /* in codes, counted from the foot of the binade's own spacing: 23 bits are held, the lowest 20 are dropped */
    const double units = floor(a / pow2(f - bias - 23)) / 1048576.0;
    int c = (int)(units + up) + (f - 1) * 8;
    if (c > top) c = top;
    if (!first && x > 0.0f && c < 1) c = 1;
    return (uint8_t)(c | sign);
}

static uint32_t mix(uint32_t x) {
    x = (x ^ (x >> 16)) * 0x9E3779B1u;
    x = (x ^ (x >> 15)) * 0x85157AF5u;
    return x ^ (x >> 16);
}

static void adam8_shard(const ElxChunkDesc* d, int index, const ElxSeg* segs, const ElxHyper* hyper, int n_groups,
                        ElxCtl* ctl) {
    uint8_t *sm = (uint8_t*)d->exp_avg, *sv = (uint8_t*)d->exp_avg_sq;
    uint8_t *em = sm + exps_at(d->n_shard), *ev = sv + exps_at(d->n_shard);
    for (int64_t b = 0; b < blocks_of(d->n_shard) && !ctl->skip; ++b) {
        const int64_t e0 = b * ELX_MOMENT_BLOCK;
        const int len = (int)(d->n_shard - e0 < ELX_MOMENT_BLOCK ? d->n_shard - e0 : ELX_MOMENT_BLOCK);
        float m[ELX_MOMENT_BLOCK], v[ELX_MOMENT_BLOCK];
        int touched = 0;
        for (int i = 0; i < len; ++i) {
            m[i] = code_value(sm[e0 + i], em[b], 1);
            v[i] = code_value(sv[e0 + i], ev[b], 0);
        }
        for (int s = d->seg_first; s < d->seg_first + d->seg_count; ++s) {
            if (segs[s].group < 0 || segs[s].group >= n_groups) continue;
            const ElxHyper h = hyper[segs[s].group];
            for (int64_t e = segs[s].begin > e0 ? segs[s].begin : e0; e < segs[s].end && e < e0 + len; ++e) {
                const int i = (int)(e - e0);
                const float om1 = 1.0f - h.beta1, om2 = 1.0f - h.beta2;
                const void* src = grad_of(d);
                float g = d->dtype == ELX_F32    ? ((const float*)src)[e]
                          : d->dtype == ELX_F16 ? orc_f16_to_f32(((const uint16_t*)src)[e])
                                                : orc_bf16_to_f32(((const uint16_t*)src)[e]);
                if (ctl->div_scale > 0.0f) g = g / ctl->div_scale;
                const float p = d->master[e];
                if (!h.adamw_mode) g = (float)((double)h.weight_decay * p + (double)g);
                const float m1 = h.beta1 * m[i], m2 = om1 * g, v1 = h.beta2 * v[i], v2 = om2 * g, v3 = v2 * g;
                m[i] = m1 + m2;
                v[i] = v1 + v3;
                /* the parameter's own step, in double */
                double bc1 = 1.0, bc2 = 1.0;
                if (h.bias_correction) {
                    double t1 = 1.0, t2 = 1.0;
                    for (int t = 0; t < ctl->step; ++t) {
                        t1 *= h.beta1;
                        t2 *= h.beta2;
                    }
                    bc1 -= t1;
                    bc2 -= t2;
                }
                double upd = m[i] / bc1 / (sqrt(v[i] / bc2) + h.eps);
                if (h.adamw_mode) upd += (double)h.weight_decay * p;
                d->master[e] = (float)(p - h.lr * upd);
                touched = 1;
            }
        }
        if (!touched) continue;
        em[b] = block_exp(m, len);
        ev[b] = block_exp(v, len);
        if (em[b] == 255 || ev[b] == 255) {
            ctl->late_inf = 1;
            ctl->status |= ELX_STAT_LATE_INF;
        }
        uint32_t key = mix((uint32_t)ctl->step * 0x632BE5ABu + (uint32_t)index * 0x9E3779B1u + 0x2545F491u);
        key = mix(mix(key ^ (uint32_t)b) ^ (uint32_t)((uint64_t)b >> 32));
        for (int i = 0; i < len; ++i) {
            const uint32_t r = mix(key + (uint32_t)i * 0x9E3779B1u);
            sm[e0 + i] = code_of(m[i], em[b], 1, (r & 0xFFFFu) / 65536.0);
            sv[e0 + i] = code_of(v[i], ev[b], 0, (r >> 16) / 65536.0);
        }
    }
    orc_cast(d->master, d->grad_param, d->dtype, d->n_shard);
}

int elx_adam8_multi(const ElxChunkDesc* descs, int first, int count, int64_t n_tiles, int dtype, const ElxSeg* segs,
                    const ElxHyper* hyper, int n_groups, ElxCtl* ctl, void* stream) {
    (void)n_tiles;
    (void)stream;
    if (!descs || !ctl) return ELX_ERR_NULL;
    if (n_groups > 64) return ELX_ERR_CAPACITY;
    for (int c = first; c < first + count; ++c) {
        if (descs[c].dtype != dtype) {
            ctl->status |= ELX_STAT_BAD_DESC;
            continue;
        }
        adam8_shard(&descs[c], c, segs, hyper, n_groups, ctl);
    }
    return ELX_OK;
}

int elx_moments_pack(const float* exp_avg, const float* exp_avg_sq, int64_t n, void* state_m, void* state_v, void* stream) {
    (void)stream;
    if (!exp_avg || !exp_avg_sq || !state_m || !state_v) return ELX_ERR_NULL;
    if (n < 0) return ELX_ERR_SIZE;
    for (int k = 0; k < 2; ++k) {
        const float* x = k ? exp_avg_sq : exp_avg;
        uint8_t* s = (uint8_t*)(k ? state_v : state_m);
        for (int64_t b = 0; b < blocks_of(n); ++b) {
            const int64_t e0 = b * ELX_MOMENT_BLOCK;
            const int len = (int)(n - e0 < ELX_MOMENT_BLOCK ? n - e0 : ELX_MOMENT_BLOCK);
            const uint8_t e = block_exp(x + e0, len);
            s[exps_at(n) + b] = e;
            for (int i = 0; i < len; ++i) s[e0 + i] = code_of(x[e0 + i], e, !k, 0.5);
        }
        const int64_t end = exps_at(n) + blocks_of(n);
        if (n) memset(s + n, 0, (size_t)(exps_at(n) - n));
        memset(s + end, 0, (size_t)(elx_moment_state_bytes(n) - end));
    }
    return ELX_OK;
}

int elx_moments_unpack(const void* state_m, const void* state_v, int64_t n, int dtype, void* exp_avg, void* exp_avg_sq,
                       void* stream) {
    (void)stream;
    if (!state_m || !state_v || !exp_avg || !exp_avg_sq) return ELX_ERR_NULL;
    if (dtype != ELX_F32 && dtype != ELX_BF16) return ELX_ERR_DTYPE;
    if (n < 0) return ELX_ERR_SIZE;
    for (int k = 0; k < 2; ++k) {
        const uint8_t* s = (const uint8_t*)(k ? state_v : state_m);
        void* out = k ? exp_avg_sq : exp_avg;
        for (int64_t i = 0; i < n; ++i) {
            const float x = code_value(s[i], s[exps_at(n) + i / ELX_MOMENT_BLOCK], !k);
            if (dtype == ELX_F32) ((float*)out)[i] = x;
            else orc_cast(&x, (uint16_t*)out + i, ELX_BF16, 1);
        }
    }
    return ELX_OK;
}

/* The operators of the wrapped model have no host-memory form: CPU tensors stay with torch. */
int elx_layer_norm_forward(const void* x, const void* weight, const void* bias, int dtype, int64_t rows, int64_t cols,
                           float eps, void* y, float* mean, float* rstd, void* stream) {
    (void)x; (void)weight; (void)bias; (void)dtype; (void)rows; (void)cols; (void)eps; (void)y; (void)mean; (void)rstd;
    (void)stream;
    return ELX_ERR_NODEVICE;
}
int64_t elx_layer_norm_backward_workspace(int64_t rows, int64_t cols) {
    (void)rows; (void)cols;
    return ELX_ERR_NODEVICE;
}
int elx_layer_norm_backward(const void* dy, const void* x, const void* weight, const float* mean, const float* rstd, int dtype,
                            int64_t rows, int64_t cols, void* dx, void* dweight, void* dbias, void* workspace,
                            int64_t workspace_bytes, void* stream) {
    (void)dy; (void)x; (void)weight; (void)mean; (void)rstd; (void)dtype; (void)rows; (void)cols; (void)dx; (void)dweight;
    (void)dbias; (void)workspace; (void)workspace_bytes; (void)stream;
    return ELX_ERR_NODEVICE;
}
int elx_embedding_forward(const void* tokens, int index_bytes, int64_t n, const void* weight, int dtype, int64_t vocab,
                          int64_t width, float scale, void* out, void* stream) {
    (void)tokens; (void)index_bytes; (void)n; (void)weight; (void)dtype; (void)vocab; (void)width; (void)scale; (void)out;
    (void)stream;
    return ELX_ERR_NODEVICE;
}
int64_t elx_embedding_backward_workspace(int64_t n, int64_t width) {
    (void)n; (void)width;
    return ELX_ERR_NODEVICE;
}
int elx_embedding_backward(const void* tokens, int index_bytes, int64_t n, const void* dout, int dtype, int64_t vocab,
                           int64_t width, float scale, int64_t padding_idx, void* dweight, void* workspace,
                           int64_t workspace_bytes, void* stream) {
    (void)tokens; (void)index_bytes; (void)n; (void)dout; (void)dtype; (void)vocab; (void)width; (void)scale;
    (void)padding_idx; (void)dweight; (void)workspace; (void)workspace_bytes; (void)stream;
    return ELX_ERR_NODEVICE;
}
