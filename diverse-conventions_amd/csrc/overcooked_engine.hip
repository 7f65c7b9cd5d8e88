// overcooked_engine.hip -- MI355X (gfx950) Overcooked rollout engine: kernels + C ABI.
//
// What it replaces: the reference's Madrona simulation of the Overcooked MDP
// (/root/reference/src/overcooked2_env/sim.cpp: 13 task-graph nodes per step, :649-688) and its
// Manager/bindings (mgr.cpp, bindings.cpp).  Semantics follow the reference's *Python* twin
// (envs/overcooked2_reimplement.py, DummyMDP) which SURVEY.md 8(a) makes normative; reference
// line numbers below are of that file unless another file is named.
//
// Execution model (see DESIGN.md for the roofline argument):
//   * one 64-lane wavefront (= one workgroup) walks groups of KPW consecutive kitchens in a
//     grid-stride loop; the next group's state records and actions are prefetched into registers
//     while the current group is processed, and the current group's plane stores drain while the
//     next group is computed (without this every wave of the chip sits in the same phase);
//   * state records are flat-copied HBM -> LDS with 16-byte loads (odd LDS stride per kitchen so
//     lane-per-kitchen accesses are bank-conflict free);
//   * phase T (lane = kitchen): the serial joint transition -- interacts in player order, moves,
//     collision rule, timestep/horizon, auto-reset -- entirely on LDS/registers;
//   * phase E (lane = tile): pot timers, reset clearing, and the 20-channel encoding of every tile
//     for both viewers, 5 dwords per (tile, viewer) staged in LDS in *output* order;
//   * flush: the staged planes leave as 16-byte-per-lane, 1 KiB-per-wave coalesced stores; the
//     state block goes back the same way.  No atomics, no inter-workgroup traffic.
//
// This file is the product path.  It never calls into oracle/ and has no CPU fallback.

#include <hip/hip_runtime.h>
#include <dlfcn.h>
#include <hip/hiprtc.h>

#include <sys/stat.h>
#include <sys/types.h>
#include <unistd.h>

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <exception>
#include <new>
#include <map>
#include <mutex>
#include <string>
#include <vector>

#include "overcooked_hip.h"
#include "overcooked_experiments.h"
#include "overcooked_debug.h"
#include "oc_internal.h"

#include "oc_step_kernel.h"
#include "oc_np_kernels.h"

// text of oc_step_common.h / oc_step_body.h (oc_step_common_src, oc_step_body_src), generated by the build
// (native.build) for the hiprtc path
#include "oc_step_kernel_src.inc"

namespace {

using namespace oc_dev;

// Per-engine specialised build of the step kernel (hiprtc): entry points by (STEP, ACT64, VEC16)
// (16-byte stores only: OC_DWORD_STORES=1, a diagnostic, runs on the ahead-of-time generic kernels).  The engine's module
// holds the first JIT_NMAIN; the four fused-rollout entries live in a module of their own, built on the first rollout
// (hiprtc time grows with the number of entry points: 14 in one module took ~3.5 s per layout, these six ~1.5 s).
enum { JIT_STEP_I32_V16, JIT_STEP_I64_V16, JIT_STEP_I32_V16_NT, JIT_STEP_I64_V16_NT, JIT_STEP_I32_V16_PL, JIT_STEP_I64_V16_PL, JIT_OBS_V16, JIT_OBS_BATCH_V16, JIT_NMAIN,
       JIT_ROLLOUT_I32 = JIT_NMAIN, JIT_ROLLOUT_I64, JIT_ROLLOUT_I32_NT, JIT_ROLLOUT_I64_NT, JIT_STEP_I32_V16_2P, JIT_STEP_I64_V16_2P, JIT_NFUNC };
const char *const kJitNames[JIT_NFUNC] = {"oc_jit_step_i32_v16", "oc_jit_step_i64_v16", "oc_jit_step_i32_v16_nt",
                                         "oc_jit_step_i64_v16_nt", "oc_jit_step_i32_v16_pl", "oc_jit_step_i64_v16_pl", "oc_jit_observe_v16", "oc_jit_observe_batch_v16",
                                         "oc_jit_rollout_i32", "oc_jit_rollout_i64", "oc_jit_rollout_i32_nt",
                                         "oc_jit_rollout_i64_nt", "oc_jit_step_i32_v16_2p", "oc_jit_step_i64_v16_2p"};
// one launch over several engines (oc_group_*): entry points of the group module
enum { GJIT_STEP_I32, GJIT_STEP_I64, GJIT_STEP_I32_NT, GJIT_STEP_I64_NT, GJIT_STEP_I32_PL, GJIT_STEP_I64_PL, GJIT_OBS, GJIT_NFUNC };
const char *const kGroupJitNames[GJIT_NFUNC] = {"oc_jit_group_step_i32", "oc_jit_group_step_i64", "oc_jit_group_step_i32_nt",
                                               "oc_jit_group_step_i64_nt", "oc_jit_group_step_i32_pl", "oc_jit_group_step_i64_pl",
                                               "oc_jit_group_observe"};
// The kitchen count stays a runtime argument, so one build serves every engine of a layout/tuning:
// compiled code objects are cached per option string for the life of the process.
// Per-XCD group sizes of the one-launch-per-step entry points of a single engine (oc_step_body.h, OC_XW_SUM): w[x] kitchens in the
// groups of XCD x, at most the tuning's kitchens per group (which sizes LDS and the state registers); sum 0: equal groups.
struct XcdWeights { int w[8]; int sum; };

struct JitModule {
    XcdWeights xw = {};                        // what the module's step / observe entry points were built with
    int halo_r = 0;                            // OC_HALO_R of the module (fresh destinations of an engine whose second plane is off a 64-byte boundary)
    int wg = 1;                                // wavefronts per workgroup of those entry points (experiment: OC_WG_WAVES)
    hipModule_t mod = nullptr;
    hipFunction_t fn[JIT_NFUNC] = {};
    int kpw = 0, gpasses = 0;
    int failed_kpw = 0, failed_gpasses = 0;    // geometry whose build failed: not tried again (the generic kernel serves)
};

// every kitchen to the standard start state (ref:387-391): empty tiles, players at their start
// tiles facing NORTH with empty hands, timestep 0.
__global__ void oc_fill_start_kernel(uint4 *state, int64_t first, int64_t count, int recq, int S, uint32_t start_posor) {
    const int64_t c = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (c >= count * recq) return;
    const int r = static_cast<int>(c % recq);
    uint32_t w[4] = {0, 0, 0, 0};
    const int idx = S - 4 * r;                 // dword S holds posor
    if (idx >= 0 && idx < 4) w[idx] = start_posor;
    state[first * recq + c] = make_uint4(w[0], w[1], w[2], w[3]);
}

// per-kitchen episode control for staggered (mixed-play style) schedules, SURVEY 8(f4):
// mask[k] != 0 -> kitchen k back to the start state; ts != NULL -> timestep[k] := ts[k] (clamped to 0..horizon-1)
__global__ void oc_episode_control_kernel(uint4 *state, int64_t n, int recq, int S, uint32_t start_posor, int horizon,
                                          const int32_t *mask, const int32_t *ts) {
    const int64_t c = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (c >= n * recq) return;
    const int64_t k = c / recq;
    const int r = static_cast<int>(c - k * recq);
    const bool reset = mask && mask[k] != 0;
    if (!reset && !(ts && r == (S + 3) / 4)) return;
    uint4 q = state[c];
    uint32_t w[4] = {q.x, q.y, q.z, q.w};
    for (int j = 0; j < 4; ++j) {
        const int idx = 4 * r + j;                      // dword index in the record
        if (reset) w[j] = idx == S ? start_posor : 0u;
        if (ts && idx == S + 3) w[j] = static_cast<uint32_t>(min(max(ts[k], 0), horizon - 1));
    }
    state[c] = make_uint4(w[0], w[1], w[2], w[3]);
}

// Checked device-to-device import (checkpoint reload without a host pass over the records): one thread per record
// validates what the kernels index with -- players on interior tiles with orientations 0..3, object names 0..4 on
// every tile and in every hand -- for either record format (P = 2: packed posor; other player counts: one word per
// player, oc_np_kernels.h); rejected records are counted.  `copy`: a record that passes is copied (oc_import_states_checked);
// otherwise nothing is written (oc_validate_states: the all-or-nothing first pass of a checkpoint reload).
__global__ void oc_import_checked_kernel(uint4 *dst, const uint4 *src, int64_t n, int recq, int S, int W, int H, int P, int copy, int32_t *n_bad) {
    const int64_t k = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (k >= n) return;
    const uint32_t *w = reinterpret_cast<const uint32_t *>(src + k * recq);
    bool ok = true;
    for (int t = 0; t < S; ++t) ok = ok && (w[t] & 0xff) <= O_SOUP;
    auto interior = [&](int p) { const int x = p % W, y = p / W; return p < S && x > 0 && y > 0 && x < W - 1 && y < H - 1; };
    if (P == 2) {
        const uint32_t posor = w[S];
        ok = ok && interior(posor & 0xff) && interior((posor >> 16) & 0xff) && ((posor >> 8) & 0xff) <= 3 && (posor >> 24) <= 3;
        ok = ok && (w[S + 1] & 0xff) <= O_SOUP && (w[S + 2] & 0xff) <= O_SOUP;
    } else {
        for (int i = 0; i < P; ++i) {
            const uint32_t pp = w[S + i];
            ok = ok && interior(pp & 0xff) && (pp >> 8) <= 3 && (w[S + P + i] & 0xff) <= O_SOUP;
        }
    }
    if (!ok) { atomicAdd(n_bad, 1); return; }
    if (copy)
        for (int q = 0; q < recq; ++q) dst[k * recq + q] = src[k * recq + q];
}

// ------------------------------------------------------------------------------------------------
// host side
thread_local char g_err[512] = "";

int fail(int code, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
    return code;
}

#define OC_HIP(call)                                                                              \
    do {                                                                                          \
        hipError_t err__ = (call);                                                                \
        if (err__ != hipSuccess)                                                                  \
            return fail(OC_ERR_HIP, "%s failed: %s (%s:%d)", #call, hipGetErrorString(err__), __FILE__, __LINE__); \
    } while (0)

}  // namespace

// error text for the other translation units of the library (rollout_ops.hip, policy_ops.hip)
int oc_internal_fail(int code, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
    return code;
}

struct oc_engine {
    oc_layout_params params;
    int64_t n;
    int device;
    int S, recq;
    int n_pots, n_counters, uniform_time;
    int pots4[4];
    uint32_t start_posor;
    int kpw, gpasses, kpp, waves_per_cu, num_cus, ablate;
    bool np_path;               // P != 2: the N-player group kernel (oc_np_kernels.h)
    int P, recd;                // players; dwords per state record
    uint32_t start_pp[4];       // N-player start entries: position | NORTH<<8
    int cu_budget;              // > 0: launches are sized for this many CUs (the stream is CU-masked), else for num_cus
    uint4 *d_state;
    uint4 *d_state_alt = nullptr;              // second record block of launches whose groups read a neighbour's kitchen (halo_launch)
    int wg_waves = 1;                          // wavefronts per workgroup of the per-engine step / observe entry points (prepare_engine: 8 on small batches)
    bool state_pinned = false;                 // a launch of this engine has been captured into a graph: d_state never moves again (note_stream)
    bool alt_failed = false;                   // the second block could not be allocated: halo launches run without halo kitchens
    DevTables *d_tabs;
    unsigned long long *d_trace;
    hipEvent_t ev0, ev1;
    JitModule jit;
    JitModule jit_fused;        // rollout entries only, built on first use for the fused rollout's own geometry
    int first_passes;           // of a group's first flush (Tuning::first)
    int encode_ilp4;            // Tuning::ilp4
    JitModule jit_fresh;        // the two step entries for fresh (time-major) destinations, built on first use for fresh_tuning()
    JitModule jit_batch;        // the batched featurisation entry with the large-batch geometry, for engines whose own geometry is a small batch's
    JitModule jit_2p;           // the in-place step entries that take the two players' actions as two buffers (oc_step_players), built on first use
    bool tuned_by_user;         // oc_set_tuning was called: its geometry then serves every kernel
    const int8_t *last_obs;
    bool planes_read_next;      // oc_internal_planes_read_next: a fresh slot's planes are read by the launch that follows (plain stores)
    int32_t *d_fold_ws;         // fold groups' arrival counters | expected counts (oc_internal_fold_workspace), or NULL
    StepArgs *d_fold_args;      // device copy of the fold step arguments (pointers to the caller's buffers NULL)
    char arch[64];
    char jit_status[256];
};

namespace {

// launch geometry of one engine inside one launch: its own (oc_set_tuning) or the one a group chose for it
struct Tuning {
    int kpw, gpasses, kpp;
    int first = 0;      // passes of a group's FIRST flush (specialised builds; 0: gpasses) -- a shorter one starts the store stream earlier
    int ilp4 = 0;       // phase E with four tiles per lane in flight where a flush has four passes (specialised builds)
};

size_t lds_bytes(const oc_engine *e, int kpw, int gpasses) {
    const int lstride = 4 * e->recq + 1;
    return sizeof(uint32_t) * (static_cast<size_t>(lds_table_dwords(e->S, e->n_pots, e->n_counters)) + kpw * kKd +
                               16 + align4(kpw * lstride) + 2 * gpasses * kWave * kTileDwords);
}

int launch_cus(const oc_engine *e) { return e->cu_budget > 0 && e->cu_budget < e->num_cus ? e->cu_budget : e->num_cus; }

StepArgs make_args(const oc_engine *e, const Tuning &tu, uint4 *state, int64_t n, const void *actions, int8_t *obs, int32_t *reward,
                   int32_t *done) {
    StepArgs a;
    a.state = state;
    a.tabs = e->d_tabs;
    a.actions = actions;
    a.actions1 = nullptr;
    a.obs = obs;
    a.reward = reward;
    a.done = done;
    a.n_kitchens = n;
    a.obs_player_stride = n * e->S * kChannels;
    a.W = e->params.width;
    a.S = e->S;
    a.recq = e->recq;
    a.lstride = 4 * e->recq + 1;
    a.kpw = tu.kpw;
    a.gpasses = tu.gpasses;
    a.kpp = tu.kpp;
    a.n_groups = static_cast<int32_t>((n + tu.kpw - 1) / tu.kpw);
    a.horizon = e->params.horizon;
    a.placement_rew = e->params.placement_in_pot_rew;
    a.dish_rew = e->params.dish_pickup_rew;
    a.soup_rew = e->params.soup_pickup_rew;
    a.n_pots = e->n_pots;
    a.n_counters = e->n_counters;
    for (int i = 0; i < 4; ++i) a.pots4[i] = e->pots4[i];
    {
        const unsigned long long w = static_cast<unsigned char>(e->params.width), mw = static_cast<unsigned char>(-e->params.width);
        a.delta_pack = mw | (w << 8) | (1ull << 16) | (0xFFull << 24);
    }
    a.uniform_time = e->uniform_time;
    a.start_posor = e->start_posor;
    a.n_steps = 1; a.tape_steps = 1;
    a.action_step_stride = 0; a.obs_step_stride = 0; a.reward_step_stride = 0; a.done_step_stride = 0;
    a.rng_seed = 0; a.rng_t0 = 0;
    a.batch_groups = a.n_groups; a.state_batch_stride = 0; a.obs_batch_stride = 0;
    a.rec_out = nullptr; a.rec_step_stride = 0;
    a.state_out = nullptr;
    a.ablate = e->ablate;
    a.trace = e->d_trace;
    return a;
}

Tuning own_tuning(const oc_engine *e) { return Tuning{e->kpw, e->gpasses, e->kpp, e->first_passes, e->encode_ilp4}; }

StepArgs make_args(const oc_engine *e, uint4 *state, int64_t n, const void *actions, int8_t *obs, int32_t *reward, int32_t *done) {
    return make_args(e, own_tuning(e), state, n, actions, obs, reward, done);
}

// Kitchen-aligned passes (opt-in, OC_ALIGNED_PASSES=1): usable when few lanes idle (>= 58 of 64 busy) and
// every flush group of `gpasses` passes still starts on a 16-byte boundary of the viewer plane.  Measured
// on cramped_room: the shorter set-up (-0.3 us to first store) is outweighed by the 11th pass and the
// partly filled wave stores (13.42 vs 13.23 us), so flat passes are the default.
int kpp_for(int S, int gpasses) {
    const char *m = OC_DIAG_ENV("OC_ALIGNED_PASSES");
    if (!m || !m[0] || m[0] == '0') return 0;
    if (S > kWave) return 0;
    const int kpp = kWave / S;
    if (kpp * S < 58) return 0;
    if ((gpasses * kpp * S * 5) % 4) return 0;
    return kpp;
}

int qn_for(int kpw, int recq) {
    const int q = (kpw * recq + kWave - 1) / kWave;      // 16-byte state chunks per lane per group
    return q <= 2 ? 2 : q >= kMaxQ ? kMaxQ : q;
}

// ---- run-time specialisation -----------------------------------------------------------------------------
// The program text handed to hiprtc pins every engine constant (the KP_* macros of oc_step_common.h) with
// #defines in front of an #include of the kernel body; a group module repeats that once per distinct layout,
// each in its own namespace, and adds entry points that dispatch a sub-range of the grid to each.
const char *const kLayoutMacros[] = {"OC_S", "OC_RECQ", "OC_KPW", "OC_GP", "OC_KPP", "OC_HORIZON", "OC_DISH_REW", "OC_NPOTS",
                                     "OC_NCOUNTERS", "OC_UNIFORM_TIME", "OC_POT0", "OC_POT1", "OC_POT2", "OC_POT3",
                                     "OC_START_POSOR", "OC_DELTA_PACK", "OC_XW_SUM", "OC_XW_PACK", "OC_XW_PREFIX", "OC_FIRST_PASSES", "OC_ENCODE_ILP4", "OC_HALO_R", "OC_GROUP_K"};

XcdWeights xcd_weights(const oc_engine *e, const Tuning &tu) {
    XcdWeights x{};
    int w[8];
    const char *m = OC_DIAG_ENV("OC_XCC_WEIGHTS");                  // experiment: "w0,...,w7"
    if (m && sscanf(m, "%d,%d,%d,%d,%d,%d,%d,%d", w, w + 1, w + 2, w + 3, w + 4, w + 5, w + 6, w + 7) == 8) {
        int sum = 0;
        for (int i = 0; i < 8; ++i) {
            if (w[i] < 0 || w[i] + 1 > tu.kpw) return x;            // LDS and the state registers hold the group's kitchens and one halo kitchen
            sum += w[i];
        }
        if (sum < 8 || sum > 255 || e->S < 16) return x;            // (one halo kitchen covers the 15 tiles in front of a group: S >= 16)
        for (int i = 0; i < 8; ++i) x.w[i] = w[i];
        x.sum = sum;
    }
    return x;
}
// OC_HALO_R of the module for fresh destinations (oc_step_body.h): 1 when a viewer plane of this engine can start off a 64-byte
// boundary -- its planes, n kitchens x S tiles x 20 bytes each, are no multiple of 64 bytes, so the second viewer's plane and every
// other time-major slot are -- and the group size is one whose own byte ranges are multiples of 64.  The kernel then reads the offsets
// off the pointers of each launch.
int halo_r_for(const oc_engine *e, const Tuning &tu) {
    if (e->np_path || e->S < 16 || (tu.kpw * e->S) % 16 || tu.kpp) return 0;
    return (e->n * e->S * kChannels) % 64 != 0 ? 1 : 0;
}
constexpr size_t kHaloCarryBytes = 2 * 16 * kTileDwords * sizeof(uint32_t);

// Wavefronts per workgroup of the per-engine step / observe entry points: the body runs as wavefront w of the workgroup on its own
// slice of the dynamic LDS (no workgroup barrier anywhere in it).  One for large batches (round 4: 11.23 / 11.26 against 11.05 us at
// 65 536 kitchens with two / four); EIGHT for the small batches an 8-GPU job runs per GPU (round 6, prepare_engine): a launch of
// 2048 one-wavefront workgroups spends ~0.5 us dealing them out, 256 workgroups of eight start together.  OC_WG_WAVES (diagnostics
// build) overrides.  Never more than fit 64 KB of LDS.
int wg_waves_for(const oc_engine *e, const Tuning &tu) {
    const char *v = OC_DIAG_ENV("OC_WG_WAVES");
    int w = v ? atoi(v) : e->wg_waves;
    if (w != 2 && w != 4 && w != 8) w = 1;
    while (w > 1 && static_cast<size_t>(w) * lds_bytes(e, tu.kpw, tu.gpasses) > 64 * 1024) w /= 2;
    return w;
}
int64_t xcd_groups(const XcdWeights &x, int64_t n) { return 8 * ((n + x.sum - 1) / x.sum); }

std::string layout_defines(const oc_engine *e, const Tuning &tu, bool per_xcd = false, int halo_r = 0) {
    char buf[128];
    std::string o;
    if (halo_r) { snprintf(buf, sizeof(buf), "#define OC_HALO_R %d\n#define OC_GROUP_K %d\n", halo_r, tu.kpw); o += buf; }
    if (per_xcd) {
        const XcdWeights x = xcd_weights(e, tu);
        if (x.sum) {
            unsigned long long pack = 0, prefix = 0;
            for (int i = 0, run = 0; i < 8; run += x.w[i], ++i) { pack |= static_cast<unsigned long long>(x.w[i]) << (8 * i); prefix |= static_cast<unsigned long long>(run) << (8 * i); }
            snprintf(buf, sizeof(buf), "#define OC_XW_SUM %d\n#define OC_XW_PACK %lluull\n", x.sum, pack); o += buf;
            snprintf(buf, sizeof(buf), "#define OC_XW_PREFIX %lluull\n", prefix); o += buf;
        }
    }
    auto def = [&](const char *name, long long v) { snprintf(buf, sizeof(buf), "#define %s %lld\n", name, v); o += buf; };
    def("OC_S", e->S);
    def("OC_RECQ", e->recq);
    def("OC_KPW", tu.kpw + (halo_r ? 1 : 0));           // (sizes LDS and the state registers: with a halo kitchen, one more than a group owns)
    def("OC_GP", tu.gpasses);
    { const char *fp = OC_DIAG_ENV("OC_FIRST_PASSES"); def("OC_FIRST_PASSES", fp ? atoi(fp) : tu.first); }   // (the environment: experiments)
    { const char *i4 = OC_DIAG_ENV("OC_ENCODE_ILP4"); def("OC_ENCODE_ILP4", i4 ? atoi(i4) : tu.ilp4); }
    def("OC_KPP", tu.kpp);
    def("OC_HORIZON", e->params.horizon);
    def("OC_DISH_REW", e->params.dish_pickup_rew);
    def("OC_NPOTS", e->n_pots);
    def("OC_NCOUNTERS", e->n_counters);
    def("OC_UNIFORM_TIME", e->uniform_time);
    def("OC_POT0", e->pots4[0]); def("OC_POT1", e->pots4[1]); def("OC_POT2", e->pots4[2]); def("OC_POT3", e->pots4[3]);
    snprintf(buf, sizeof(buf), "#define OC_START_POSOR %uu\n", e->start_posor); o += buf;
    const unsigned long long w = static_cast<unsigned char>(e->params.width), mw = static_cast<unsigned char>(-e->params.width);
    snprintf(buf, sizeof(buf), "#define OC_DELTA_PACK %lluull\n", mw | (w << 8) | (1ull << 16) | (0xFFull << 24)); o += buf;
    return o;
}

// Store mode of the plane stores per destination kind (store16 in oc_step_common.h); OC_STORE_MODE="a,b" overrides
// (a: destination overwritten in place, b: a fresh slot every step) for experiments.  Measured on MI355X
// (profiles/r02_store_modes.log), us per launch plain / nt / sc1: cramped_room 65 536 kitchens in place 13.47 / 13.62 /
// 12.21, into time-major slots - / 13.58 / 14.27; five layouts x 8192 in one launch 14.29 / 16.08 / 13.15.  Fresh slots
// with the round-3 geometry, nt / sc1 nt: 12.69 / 12.50 (profiles/r03_ab_time_major_sc1nt.log).
int store_mode_env(int which, int dflt) {
    const char *m = OC_DIAG_ENV("OC_STORE_MODE");
    int a = -1, b = -1;
    if (m && sscanf(m, "%d,%d", &a, &b) == 2 && a >= 0 && a <= 4 && b >= 0 && b <= 4) return which == 0 ? a : b;
    return dflt;
}
int store_mode_in_place() { return store_mode_env(0, SM_SC1); }
int store_mode_fresh() { return store_mode_env(1, SM_SC1_NT); }
std::string sm1f_batch(int sm) {
    char b[48];
    snprintf(b, sizeof(b), ", %d, false, true", sm);
    return b;
}

// Kernel-argument preload: the leading scalar arguments of an entry point (14 dwords: six pointers and the kitchen count) arrive in
// SGPRs with the wavefront instead of through s_load (gfx950 firmware under ROCm 7 honours it: tools/probes/kernarg_preload.hip; the
// compiler keeps a compatibility prologue that loads them the old way).  Part of the program text, so that it is part of the cache key.
constexpr const char *kJitPreloadOption = "-amdgpu-kernarg-preload-count=14";

std::string jit_prologue() {
    std::string t = std::string("// hiprtc options: -O3 -std=c++17 -packed-fp32-ops -mllvm ") + kJitPreloadOption + "\n#define OC_JIT 1\n";
    if (const char *nu = OC_DIAG_ENV("OC_NOUNROLL")) t += std::string("#define OC_NOUNROLL ") + ((nu[0] && nu[0] != '0') ? "1\n" : "0\n");
    // (batched flush: on by default for grids of at most 32 tiles, see oc_step_body.h; the environment overrides)
    if (const char *ff = OC_DIAG_ENV("OC_FAST_FLUSH")) t += std::string("#define OC_FAST_FLUSH ") + ((ff[0] && ff[0] != '0') ? "1\n" : "0\n");
    if (const char *tr = OC_DIAG_ENV("OC_JIT_TRACE")) t += std::string("#define OC_TRACE ") + ((tr[0] && tr[0] != '0') ? "1\n" : "0\n");   // diagnostics: keep the phase stamps
    if (const char *ab = OC_DIAG_ENV("OC_ABLATE")) t += std::string("#define OC_JIT_ABLATE ") + std::to_string(atoi(ab)) + "\n";     // diagnostics: phases skipped (timing only)
    if (const char *xr = OC_DIAG_ENV("OC_XCC_ROT")) t += std::string("#define OC_XCC_ROT ") + std::to_string(atoi(xr)) + "\n";   // experiment: rotate block -> group
    t += "#include \"oc_step_common.h\"\n";
    return t;
}

std::string jit_layout_block(const std::string &ns, const std::string &defines) {
    std::string t = "#define OC_NS " + ns + "\n" + defines + "#include \"oc_step_body.h\"\n#undef OC_NS\n";
    for (const char *m : kLayoutMacros) t += std::string("#undef ") + m + "\n";
    return t;
}

// one engine: the twelve step / observe / rollout entry points + the batched observe
// K-steps-per-launch rollouts want the geometry the per-step kernel had before the write-through stores: a wavefront's
// T phases and flushes come once per step for ALL its kitchens, so bigger groups win (32 kitchens per group on the smallest
// grids: 7.7 us per step at 65 536 kitchens against 8.2 with the per-step kernel's 16).
Tuning fused_tuning(const oc_engine *e) {
    if (e->tuned_by_user) return own_tuning(e);
    int kpw = e->recq <= 6 ? 32 : 16;
    while (kpw > 4 && kpw * e->recq > kMaxQ * kWave) kpw -= 4;
    while (kpw > 4 && kpw % 8 == 0 && e->n / kpw < 2048) kpw /= 2;
    return Tuning{kpw, 4, kpp_for(e->S, 4)};
}

// Steps whose planes go to a FRESH destination (a time-major trajectory slot: every byte to HBM) of a large batch want fewer
// store streams in flight than in-place steps: 16-kitchen groups, the plain flush loop, EIGHT persistent wavefronts per CU
// (profiles/r02_ab_time_major.log, 65 536 kitchens into 64 slots: cramped_room 12.73 us against 13.25 with twelve per CU and
// 13.49 with the in-place geometry of the smallest grids) and, since round 3, four passes per flush with write-through
// non-temporal (`sc1 nt`) plane stores (profiles/r03_ab_time_major_sc1nt.log: cramped_room 12.69 -> 12.50, coordination_ring
// 15.99 -> 15.35, counter_circuit 24.43 -> 23.55, asymmetric_advantages 28.23 -> 27.03 us; a launch that only streams the same
// bytes to fresh destinations takes 10.3 us, profiles/r03_probe_store_ceiling.log).  They run from a module of their own,
// built on the first such step.
constexpr int kFreshWavesPerCu = 8;
bool fresh_geometry_shape(const oc_engine *e) { return !e->tuned_by_user && e->kpw >= 16 && (e->n + 15) / 16 >= 3072; }
bool has_fresh_geometry(const oc_engine *e) { return e->jit.mod && fresh_geometry_shape(e); }
// (first flush of a group: two passes, one on the larger grids -- round 4, profiles/r04_ab_first_passes.log, 65 536 kitchens, us per
// launch without / with: cramped_room 12.08 / 11.93, coordination_ring 15.24 / 14.60, counter_circuit 23.34 / 22.59,
// asymmetric_advantages 26.57 / 25.89)
Tuning fresh_tuning_shape(const oc_engine *e) { return Tuning{16, 4, kpp_for(e->S, 4), e->S > 32 ? 1 : 2}; }
Tuning fresh_tuning(const oc_engine *e) { return has_fresh_geometry(e) ? fresh_tuning_shape(e) : own_tuning(e); }

enum { SRC_ALL = 0, SRC_ROLLOUT = 1, SRC_FRESH = 2, SRC_BATCH = 3, SRC_TWOPTR = 4 };
std::string jit_source_single(const oc_engine *e, const Tuning &tu, int which, int waves_per_cu);
std::string jit_source_single(const oc_engine *e) { return jit_source_single(e, own_tuning(e), SRC_ALL, e->waves_per_cu); }

std::string jit_source_single(const oc_engine *e, const Tuning &tu, int which, int waves_per_cu) {
    char buf[1536];
    const bool rollout_only = which == SRC_ROLLOUT;
    std::string t = jit_prologue();
    if ((which == SRC_FRESH || which == SRC_BATCH) && !OC_DIAG_ENV("OC_FAST_FLUSH")) t = "#define OC_FAST_FLUSH 0\n" + t;
    const bool per_xcd = which == SRC_ALL || which == SRC_FRESH || which == SRC_TWOPTR;
    const XcdWeights xw = per_xcd ? xcd_weights(e, tu) : XcdWeights{};
    const int wg = per_xcd ? wg_waves_for(e, tu) : 1;
    const int halo_r = (which == SRC_FRESH && !xw.sum && !OC_DIAG_ENV("OC_NO_HALO")) ? halo_r_for(e, tu) : 0;
    t += jit_layout_block("oc_l0", layout_defines(e, tu, per_xcd, halo_r));
    // register budget: enough waves per SIMD for the persistent-wave count to be fully resident
    const char *mw = OC_DIAG_ENV("OC_MIN_WAVES");
    const int min_waves = mw ? atoi(mw) : (waves_per_cu + 3) / 4;
    const int qn = qn_for(tu.kpw + (halo_r ? 1 : 0), e->recq);
    auto entry = [&](const char *name, const char *targs, bool batch = false) {
        // (the group count follows from the kitchen count, except for the batched featurisation whose groups run over all items:
        // derived in the entry point, it needs no scalar load in front of the first state request either)
        char ng[96] = "";
        if (!batch && xw.sum) snprintf(ng, sizeof(ng), "a.n_groups = 8 * static_cast<int>((p_n + %d) / %d); ", xw.sum - 1, xw.sum);
        else if (!batch) snprintf(ng, sizeof(ng), "a.n_groups = static_cast<int>((p_n + %d) / %d); ", tu.kpw - 1, tu.kpw);
        // The seven values every wavefront needs before it can ask memory for anything -- the buffer pointers and the kitchen count --
        // are leading scalar arguments: the build preloads them into SGPRs at wavefront launch (kJitPreloadOption), so the front
        // does not open with a scalar-memory round trip for the kernel arguments; the rest of StepArgs is constants of the build
        // or read later.  (launch_jit packs [seven scalars | StepArgs].)
        const int wgw = (per_xcd && !batch) ? wg : 1;
        char call[256];
        if (wgw > 1)
            snprintf(call, sizeof(call), "const int w_ = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); oc_dev::oc_l0::step_body<%s>(a, blockIdx.x * %d + w_, gridDim.x * %d, w_ * %d, threadIdx.x & 63);",
                     targs, wgw, wgw, static_cast<int>(lds_bytes(e, tu.kpw, tu.gpasses) / 4));
        else
            snprintf(call, sizeof(call), "oc_dev::oc_l0::step_body<%s>(a, blockIdx.x, gridDim.x);", targs);
        // (two-pointer entries, SRC_TWOPTR: player 1's action buffer as an eighth scalar behind the seven preloaded ones)
        snprintf(buf, sizeof(buf), "extern \"C\" __global__ __launch_bounds__(%d, %d) void %s(uint4 *p_state, const oc_dev::DevTables *p_tabs, "
                 "const void *p_actions, int8_t *p_obs, int32_t *p_reward, int32_t *p_done, long long p_n, %sconst oc_dev::StepArgs a0) { "
                 "oc_dev::StepArgs a = a0; a.state = p_state; a.tabs = p_tabs; a.actions = p_actions; a.obs = p_obs; a.reward = p_reward; "
                 "a.done = p_done; a.n_kitchens = p_n; %s%s%s }\n", 64 * wgw, min_waves, name, which == SRC_TWOPTR ? "const void *p_actions1, " : "",
                 which == SRC_TWOPTR ? "a.actions1 = p_actions1; " : "", ng, call);
        t += buf;
    };
    auto targs = [&](const char *step, const char *act64, const char *vec16, const char *rest) {
        char tb[256];
        snprintf(tb, sizeof(tb), "%s, %s, %s, %d%s", step, act64, vec16, qn, rest);
        return std::string(tb);
    };
    // store mode of the observation planes by destination kind (see store16): in place / fresh slot every step
    const int sm_in_place = store_mode_in_place(), sm_fresh = store_mode_fresh();
    char sm0[32], sm1[32], sm0f[48], sm1f[48];
    snprintf(sm0, sizeof(sm0), ", %d", sm_in_place); snprintf(sm1, sizeof(sm1), ", %d", sm_fresh);
    snprintf(sm0f, sizeof(sm0f), ", %d, true", sm_in_place); snprintf(sm1f, sizeof(sm1f), ", %d, true", sm_fresh);
    if (rollout_only) {
        entry("oc_jit_rollout_i32", targs("true", "false", "true", sm0f).c_str());
        entry("oc_jit_rollout_i64", targs("true", "true", "true", sm0f).c_str());
        entry("oc_jit_rollout_i32_nt", targs("true", "false", "true", sm1f).c_str());
        entry("oc_jit_rollout_i64_nt", targs("true", "true", "true", sm1f).c_str());
        return t;
    }
    // (_pl: a fresh slot whose planes the NEXT launch reads -- the policy kernel of a rollout with the policies in the loop: plain
    // stores leave them in L2 for it, and their write-back hides under that launch; oc_internal_planes_read_next)
    if (which == SRC_FRESH) {
        entry("oc_jit_step_i32_v16_nt", targs("true", "false", "true", sm1).c_str());
        entry("oc_jit_step_i64_v16_nt", targs("true", "true", "true", sm1).c_str());
        entry("oc_jit_step_i32_v16_pl", targs("true", "false", "true", ", 0").c_str());
        entry("oc_jit_step_i64_v16_pl", targs("true", "true", "true", ", 0").c_str());
        return t;
    }
    if (which == SRC_BATCH) {
        entry("oc_jit_observe_batch_v16", targs("false", "false", "true", sm1f_batch(sm_fresh).c_str()).c_str(), true);
        return t;
    }
    if (which == SRC_TWOPTR) {                                        // in-place steps whose players' actions arrive in two buffers (oc_step_players)
        char sm2[64];
        snprintf(sm2, sizeof(sm2), ", %d, false, false, false, true", sm_in_place);
        entry("oc_jit_step_i32_v16_2p", targs("true", "false", "true", sm2).c_str());
        entry("oc_jit_step_i64_v16_2p", targs("true", "true", "true", sm2).c_str());
        return t;
    }
    entry("oc_jit_step_i32_v16", targs("true", "false", "true", sm0).c_str());
    entry("oc_jit_step_i64_v16", targs("true", "true", "true", sm0).c_str());
    entry("oc_jit_step_i32_v16_nt", targs("true", "false", "true", sm1).c_str());
    entry("oc_jit_step_i64_v16_nt", targs("true", "true", "true", sm1).c_str());
    entry("oc_jit_step_i32_v16_pl", targs("true", "false", "true", ", 0").c_str());
    entry("oc_jit_step_i64_v16_pl", targs("true", "true", "true", ", 0").c_str());
    entry("oc_jit_observe_v16", targs("false", "false", "true", sm0).c_str());
    entry("oc_jit_observe_batch_v16", targs("false", "false", "true", sm1f_batch(sm_fresh).c_str()).c_str(), true);
    return t;
}

// several engines in one module: distinct layout blocks + entry points that hand each sub-range of the grid to the
// body of its segment's layout (GroupArgs in oc_step_common.h).  layout_of_seg is filled with the block index per segment.
std::string jit_source_group(const std::vector<const oc_engine *> &engines, const std::vector<Tuning> &tunings, int min_waves,
                             std::vector<int> &layout_of_seg) {
    char buf[1024];
    std::string t = jit_prologue();
    std::vector<std::string> blocks;
    std::vector<int> qn_of_block;
    layout_of_seg.clear();
    for (size_t i = 0; i < engines.size(); ++i) {
        const std::string d = layout_defines(engines[i], tunings[i]);
        size_t j = 0;
        while (j < blocks.size() && blocks[j] != d) ++j;
        if (j == blocks.size()) {
            blocks.push_back(d);
            qn_of_block.push_back(qn_for(tunings[i].kpw, engines[i]->recq));
            snprintf(buf, sizeof(buf), "oc_l%zu", j);
            t += jit_layout_block(buf, d);
        }
        layout_of_seg.push_back(static_cast<int>(j));
    }
    // The block -> segment map (segment count, first blocks, layout indices) arrives as ten leading scalar arguments, preloaded into
    // SGPRs like the per-engine entry points' pointers (kJitPreloadOption): a wavefront knows its segment without a scalar load, and
    // the one that follows -- that segment's pointers, at an offset only now known -- is the only round trip in front of its first
    // memory request (two in a row before: header, then segment).  The segment's group count is derived from its kitchen count.
    t += "template <bool STEP, bool ACT64, int SM>\n"
         "__device__ __forceinline__ void oc_group_body(const oc_dev::GroupArgs &m, int n_segs, int f1, int f2, int f3, int f4, int f5, int f6, int f7, int f8, unsigned layouts) {\n"
         "    const int b = blockIdx.x;\n"
         "    int s = 0, lo = 0, hi = f1;\n"
         "    if (1 < n_segs && b >= f1) { s = 1; lo = f1; hi = f2; }\n"
         "    if (2 < n_segs && b >= f2) { s = 2; lo = f2; hi = f3; }\n"
         "    if (3 < n_segs && b >= f3) { s = 3; lo = f3; hi = f4; }\n"
         "    if (4 < n_segs && b >= f4) { s = 4; lo = f4; hi = f5; }\n"
         "    if (5 < n_segs && b >= f5) { s = 5; lo = f5; hi = f6; }\n"
         "    if (6 < n_segs && b >= f6) { s = 6; lo = f6; hi = f7; }\n"
         "    if (7 < n_segs && b >= f7) { s = 7; lo = f7; hi = f8; }\n"
         "    const int bid = b - lo, nb = hi - lo;\n"
         "    oc_dev::StepArgs a = m.seg[s];\n"
         "    switch ((layouts >> (4 * s)) & 15u) {\n";
    for (size_t j = 0; j < blocks.size(); ++j) {
        int kpw_j = 1;
        for (size_t i = 0; i < engines.size(); ++i) if (layout_of_seg[i] == static_cast<int>(j)) kpw_j = tunings[i].kpw;
        snprintf(buf, sizeof(buf), "    case %zu: a.n_groups = static_cast<int>((a.n_kitchens + %d) / %d); oc_dev::oc_l%zu::step_body<STEP, ACT64, true, %d, SM>(a, bid, nb); break;\n",
                 j, kpw_j - 1, kpw_j, j, qn_of_block[j]);
        t += buf;
    }
    t += "    default: break;\n    }\n}\n";
    auto entry = [&](const char *name, const char *targs) {
        snprintf(buf, sizeof(buf), "extern \"C\" __global__ __launch_bounds__(64, %d) void %s(int n_segs, int f1, int f2, int f3, int f4, int f5, int f6, int f7, "
                 "int f8, unsigned layouts, int pad0, int pad1, const oc_dev::GroupArgs m) { oc_group_body<%s>(m, n_segs, f1, f2, f3, f4, f5, f6, f7, f8, layouts); }\n",
                 min_waves, name, targs);
        t += buf;
    };
    char ta[64];
    auto ts = [&](const char *step, const char *act64, int sm) { snprintf(ta, sizeof(ta), "%s, %s, %d", step, act64, sm); return ta; };
    entry("oc_jit_group_step_i32", ts("true", "false", store_mode_in_place()));
    entry("oc_jit_group_step_i64", ts("true", "true", store_mode_in_place()));
    entry("oc_jit_group_step_i32_nt", ts("true", "false", store_mode_fresh()));
    entry("oc_jit_group_step_i64_nt", ts("true", "true", store_mode_fresh()));
    entry("oc_jit_group_step_i32_pl", ts("true", "false", 0));      // (fresh slots the next launch reads: plain stores, see _pl above)
    entry("oc_jit_group_step_i64_pl", ts("true", "true", 0));
    entry("oc_jit_group_observe", ts("false", "false", store_mode_in_place()));
    return t;
}

// ---- code-object caches: per process (engines of one layout/tuning share a build) and on disk (the ranks of a
// multi-GPU job and later runs share it: 8 ranks x 5 layouts would otherwise compile the same five kernels)
uint64_t fnv1a(const std::string &s, uint64_t h) {
    for (unsigned char c : s) { h ^= c; h *= 0x100000001B3ull; }
    return h;
}

// The cache directory must be the caller's own: a code object read from it is loaded onto the GPU as the step kernel, so a
// directory somebody else could have written to (created by another user, or group / world writable) is not used at all.
std::string disk_cache_dir() {
    const char *env = getenv("OC_JIT_CACHE");               // a directory, or "0" / "off" to disable
    if (env && (!strcmp(env, "0") || !strcmp(env, "off") || !env[0])) return "";
    std::string dir;
    if (env) dir = env;
    else if (const char *x = getenv("XDG_CACHE_HOME")) dir = std::string(x) + "/overcooked_hip";
    else if (const char *h = getenv("HOME")) dir = std::string(h) + "/.cache/overcooked_hip";
    else { char b[64]; snprintf(b, sizeof(b), "/tmp/overcooked_hip-%u", static_cast<unsigned>(getuid())); dir = b; }
    // mkdir -p (failures show below: what cannot be stat'ed is not used)
    for (size_t i = 1; i <= dir.size(); ++i)
        if (i == dir.size() || dir[i] == '/') (void)mkdir(dir.substr(0, i).c_str(), 0700);
    struct stat st;
    if (stat(dir.c_str(), &st) != 0 || !S_ISDIR(st.st_mode) || st.st_uid != getuid() || (st.st_mode & (S_IWGRP | S_IWOTH))) return "";
    return dir;
}

// File = header {magic, length, checksum of the code object} + the code object; anything that does not check out is ignored
// (and overwritten by the next compile).
struct CacheHeader {
    char magic[8];
    uint64_t length, checksum;
};
const char kCacheMagic[8] = {'O', 'C', 'J', 'I', 'T', '0', '0', '2'};
uint64_t fnv1a_bytes(const char *p, size_t n) {
    uint64_t h = 0xCBF29CE484222325ull;
    for (size_t i = 0; i < n; ++i) { h ^= static_cast<unsigned char>(p[i]); h *= 0x100000001B3ull; }
    return h;
}

bool disk_cache_read(const std::string &path, std::vector<char> &code) {
    FILE *f = fopen(path.c_str(), "rb");
    if (!f) return false;
    bool ok = false;
    CacheHeader hd;
    if (fread(&hd, sizeof(hd), 1, f) == 1 && memcmp(hd.magic, kCacheMagic, 8) == 0 && hd.length > 64 && hd.length < (1ull << 28)) {
        code.resize(static_cast<size_t>(hd.length));
        ok = fread(code.data(), 1, code.size(), f) == code.size() && fgetc(f) == EOF && memcmp(code.data(), "\x7f" "ELF", 4) == 0 &&
             fnv1a_bytes(code.data(), code.size()) == hd.checksum;
    }
    fclose(f);
    if (!ok) code.clear();
    return ok;
}

void disk_cache_write(const std::string &path, const std::vector<char> &code) {
    char tmp[64];
    snprintf(tmp, sizeof(tmp), ".tmp.%d", static_cast<int>(getpid()));
    const std::string t = path + tmp;
    FILE *f = fopen(t.c_str(), "wb");
    if (!f) return;
    CacheHeader hd;
    memcpy(hd.magic, kCacheMagic, 8);
    hd.length = code.size();
    hd.checksum = fnv1a_bytes(code.data(), code.size());
    const bool ok = fwrite(&hd, sizeof(hd), 1, f) == 1 && fwrite(code.data(), 1, code.size(), f) == code.size();
    if (fclose(f) != 0 || !ok || rename(t.c_str(), path.c_str()) != 0) (void)remove(t.c_str());   // rename: whole file or nothing
}

long long g_jit_builds = 0;               // hiprtc compilations this process has run (oc_debug_jit_builds): cache misses, ~1-1.5 s each

// ---- ahead-of-time code objects (round 6).  The per-layout specialisations are hiprtc builds of program text the library generates;
// `__graft_entry__.build()` generates that text for the BASELINE shapes WITHOUT a GPU (oc_debug_aot_build: hiprtc cross-compiles) and
// leaves the code objects in <directory of this library>/aot/, named by a hash of everything they depend on (target, program text,
// both kernel headers, ABI version -- not the compiler's version: a code object is what it is whoever built it).  oc_create /
// oc_group_create / the side modules look there before the disk cache and before compiling, so a cold box loads a module in
// milliseconds instead of compiling for a second (oc_kernel_build_info: "...; ahead of time").
std::string g_aot_out;                    // non-empty while oc_debug_aot_build runs: every code object that passes through is also written here
std::string aot_dir() {
    static const std::string dir = [] {
        Dl_info info;
        if (!dladdr(reinterpret_cast<const void *>(&oc_internal_fail), &info) || !info.dli_fname) return std::string();
        const std::string lib = info.dli_fname;
        const size_t i = lib.rfind('/');
        return (i == std::string::npos ? std::string(".") : lib.substr(0, i)) + "/aot";
    }();
    return dir;
}

// Compile `text`; on success `code` holds the code object.  Needs no GPU.  `from` (optional) says where it came from.
int jit_compile_text(const std::string &text, const char *arch, std::vector<char> &code, std::string &log, const char **from = nullptr) {
    static std::mutex mu;
    static std::map<std::string, std::vector<char>> cache;
    const std::string key = std::string(arch) + "\n" + text;
    {
        std::lock_guard<std::mutex> lock(mu);
        auto it = cache.find(key);
        if (it != cache.end()) { code = it->second; if (from) *from = "process cache"; return OC_OK; }
    }
    // ahead of time: built with the library (see aot_dir)
    std::string aot_name;
    {
        char abi[32];
        snprintf(abi, sizeof(abi), "abi %d\n", OC_ABI_VERSION);
        const std::string all = std::string(abi) + key + "\n--common--\n" + oc_step_common_src + "\n--body--\n" + oc_step_body_src;
        char name[64];
        snprintf(name, sizeof(name), "/%016llx%016llx.hsaco", static_cast<unsigned long long>(fnv1a(all, 0xCBF29CE484222325ull)),
                 static_cast<unsigned long long>(fnv1a(all, 0x9E3779B97F4A7C15ull)));
        aot_name = name;
        const std::string ad = aot_dir();
        if (!ad.empty() && disk_cache_read(ad + aot_name, code)) {
            if (!g_aot_out.empty() && g_aot_out != ad) disk_cache_write(g_aot_out + aot_name, code);
            std::lock_guard<std::mutex> lock(mu);
            cache[key] = code;
            if (from) *from = "ahead of time";
            return OC_OK;
        }
    }
    // disk: the name hashes everything the code object depends on (program text, both headers, target, compiler version)
    std::string path;
    const std::string dir = disk_cache_dir();
    if (!dir.empty()) {
        int maj = 0, min = 0, rt = 0;
        (void)hiprtcVersion(&maj, &min);
        (void)hipRuntimeGetVersion(&rt);
        char ver[160];
        // compiler + runtime as exactly as they identify themselves: hiprtc's version, the runtime's, and the HIP build this
        // library was compiled against (patch level and git hash)
        snprintf(ver, sizeof(ver), "hiprtc %d.%d runtime %d built-with %d.%d.%d-%s abi %d\n", maj, min, rt, HIP_VERSION_MAJOR, HIP_VERSION_MINOR,
                 HIP_VERSION_PATCH, HIP_VERSION_GITHASH, OC_ABI_VERSION);
        const std::string all = std::string(ver) + key + "\n--common--\n" + oc_step_common_src + "\n--body--\n" + oc_step_body_src;
        char name[64];
        snprintf(name, sizeof(name), "/%016llx%016llx.hsaco", static_cast<unsigned long long>(fnv1a(all, 0xCBF29CE484222325ull)),
                 static_cast<unsigned long long>(fnv1a(all, 0x9E3779B97F4A7C15ull)));
        path = dir + name;
        if (disk_cache_read(path, code)) {
            if (!g_aot_out.empty()) disk_cache_write(g_aot_out + aot_name, code);
            std::lock_guard<std::mutex> lock(mu);
            cache[key] = code;
            if (from) *from = "disk cache";
            return OC_OK;
        }
    }
    hiprtcProgram prog = nullptr;
    const char *headers[2] = {oc_step_common_src, oc_step_body_src};
    const char *names[2] = {"oc_step_common.h", "oc_step_body.h"};
    if (hiprtcCreateProgram(&prog, text.c_str(), "oc_step_jit.hip", 2, headers, names) != HIPRTC_SUCCESS) {
        log = "hiprtcCreateProgram failed";
        return OC_ERR_HIP;
    }
    const std::string archopt = std::string("--offload-arch=") + arch;
    const char *copts[] = {archopt.c_str(), "-O3", "-std=c++17", "-mllvm", kJitPreloadOption, "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"};
    const hiprtcResult r = hiprtcCompileProgram(prog, sizeof(copts) / sizeof(copts[0]), copts);
    size_t n = 0;
    if (hiprtcGetProgramLogSize(prog, &n) == HIPRTC_SUCCESS && n > 1) { log.resize(n); hiprtcGetProgramLog(prog, &log[0]); }
    int rc = OC_OK;
    if (r != HIPRTC_SUCCESS) {
        rc = OC_ERR_HIP;
        if (log.empty()) log = hiprtcGetErrorString(r);
    } else if (hiprtcGetCodeSize(prog, &n) != HIPRTC_SUCCESS || n == 0) {
        rc = OC_ERR_HIP;
        log = "hiprtc produced no code object";
    } else {
        code.resize(n);
        hiprtcGetCode(prog, code.data());
        if (const char *dump = OC_DIAG_ENV("OC_JIT_DUMP")) {                 // diagnostics: keep the code object for llvm-objdump
            if (FILE *f = fopen(dump, "wb")) { fwrite(code.data(), 1, code.size(), f); fclose(f); }
        }
        if (!path.empty()) disk_cache_write(path, code);
        if (!g_aot_out.empty()) disk_cache_write(g_aot_out + aot_name, code);
        std::lock_guard<std::mutex> lock(mu);
        cache[key] = code;
        ++g_jit_builds;
        if (from) *from = "compiled";
    }
    hiprtcDestroyProgram(&prog);
    return rc;
}

void jit_unload(oc_engine *e) {
    if (e->jit.mod) (void)hipModuleUnload(e->jit.mod);
    e->jit = JitModule();
    if (e->jit_fused.mod) (void)hipModuleUnload(e->jit_fused.mod);
    e->jit_fused = JitModule();
    if (e->jit_fresh.mod) (void)hipModuleUnload(e->jit_fresh.mod);
    e->jit_fresh = JitModule();
    if (e->jit_batch.mod) (void)hipModuleUnload(e->jit_batch.mod);
    e->jit_batch = JitModule();
    if (e->jit_2p.mod) (void)hipModuleUnload(e->jit_2p.mod);
    e->jit_2p = JitModule();
}

bool jit_disabled(const oc_engine *e, char *status, size_t cap) {
    if (const char *off = getenv("OC_NO_JIT")) {
        if (off[0] && off[0] != '0') { snprintf(status, cap, "disabled by OC_NO_JIT"); return true; }
    }
    if (e->ablate) { snprintf(status, cap, "disabled by phase ablation (diagnostics use the generic kernel)"); return true; }
    return false;
}

// (Re)build the engine's specialised kernel for its current tuning.  Failure is not an error: the
// ahead-of-time generic kernel stays in use and jit_status says why.
void jit_build(oc_engine *e) {
    jit_unload(e);
    if (jit_disabled(e, e->jit_status, sizeof(e->jit_status))) return;
    std::vector<char> code;
    std::string log;
    const char *from = "";
    if (jit_compile_text(jit_source_single(e), e->arch, code, log, &from) != OC_OK) {
        snprintf(e->jit_status, sizeof(e->jit_status), "hiprtc: %.220s", log.c_str());
        return;
    }
    hipModule_t mod = nullptr;
    if (hipModuleLoadData(&mod, code.data()) != hipSuccess) {
        (void)hipGetLastError();
        snprintf(e->jit_status, sizeof(e->jit_status), "hipModuleLoadData failed");
        return;
    }
    JitModule j;
    j.mod = mod;
    for (int i = 0; i < JIT_NMAIN; ++i)
        if (hipModuleGetFunction(&j.fn[i], mod, kJitNames[i]) != hipSuccess) {
            (void)hipGetLastError();
            (void)hipModuleUnload(mod);
            snprintf(e->jit_status, sizeof(e->jit_status), "entry point %s missing", kJitNames[i]);
            return;
        }
    j.kpw = e->kpw;
    j.gpasses = e->gpasses;
    j.xw = xcd_weights(e, own_tuning(e));
    j.wg = wg_waves_for(e, own_tuning(e));
    e->jit = j;
    snprintf(e->jit_status, sizeof(e->jit_status), "specialised for %s (kpw %d, passes %d; %s)", e->arch, e->kpw, e->gpasses, from);
}


// Plane stores are 16 bytes per lane whatever the alignment of the caller's buffer beyond the 4 bytes the ABI asks for
// (see store16 in oc_step_common.h); OC_DWORD_STORES=1 selects the dword-store kernels instead (diagnostics).
bool wide_stores() {
    const char *v = getenv("OC_DWORD_STORES");            // read per launch so that a test can switch within one process
    return !(v && v[0] && v[0] != '0');
}

template <bool STEP, bool ACT64, bool VEC16, int QN>
void launch_q(const StepArgs &a, unsigned grid, size_t shmem, hipStream_t s) {
    hipLaunchKernelGGL((oc_step_kernel<STEP, ACT64, VEC16, QN>), dim3(grid), dim3(kWave), shmem, s, a);
}

template <bool STEP, bool ACT64, bool VEC16>
void launch_v(const StepArgs &a, unsigned grid, size_t shmem, hipStream_t s) {
    switch (qn_for(a.kpw, a.recq)) {
    case 2: launch_q<STEP, ACT64, VEC16, 2>(a, grid, shmem, s); break;
    case 3: launch_q<STEP, ACT64, VEC16, 3>(a, grid, shmem, s); break;
    case 4: launch_q<STEP, ACT64, VEC16, 4>(a, grid, shmem, s); break;
    default: launch_q<STEP, ACT64, VEC16, kMaxQ>(a, grid, shmem, s); break;
    }
}

// A launch of a module whose groups also load a kitchen they do not own (OC_HALO_R; OC_XW_SUM in the diagnostics build) must not
// write records into the block it reads them from: the owner of a halo kitchen is another wavefront of the same launch, and nothing
// orders its write-back against the neighbour's read (a reader that comes second would step the kitchen twice).  Such a launch reads
// e->d_state and writes a second block, and the two swap roles afterwards -- the state block's address is not part of the ABI, and
// every entry point takes e->d_state afresh.  A launch that is being captured into a graph cannot swap on replay: it gets no second
// block, and the kernel then runs without halo kitchens (oc_step_body.h).  -> the block to hand the kernel as state_out, or NULL.
uint4 *halo_state_out(oc_engine *e, hipStream_t s) {
    if (e->state_pinned) return nullptr;
    hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(s, &cs) != hipSuccess) { (void)hipGetLastError(); return nullptr; }
    if (cs != hipStreamCaptureStatusNone) { e->state_pinned = true; return nullptr; }
    return e->d_state_alt;                                            // (allocated with the module that needs it: ensure_halo_block)
}

// The second record block, allocated where the module that needs it is built (oc_prepare_kernels, or the first step into a fresh
// destination) -- never inside a later launch: hipMalloc synchronises the device and has no business on the step path or beside
// another stream's capture.  It doubles the engine's record memory (n kitchens x record bytes).  Without it (allocation refused) the
// module's launches run without halo kitchens -- correct, slower -- and oc_kernel_build_info says so.
void ensure_halo_block(oc_engine *e) {
    if (e->d_state_alt || e->alt_failed) return;
    if (hipMalloc(reinterpret_cast<void **>(&e->d_state_alt), static_cast<size_t>(e->n) * e->recq * sizeof(uint4)) != hipSuccess) {
        (void)hipGetLastError();
        e->d_state_alt = nullptr;
        e->alt_failed = true;
        const size_t len = strlen(e->jit_status);
        snprintf(e->jit_status + len, sizeof(e->jit_status) - len, "; no second record block: fresh destinations without halo kitchens");
    }
}

// A graph captured from ANY entry point of this engine has the record block's address in its kernel arguments, so once a launch has
// been captured the blocks must never swap again (a replay would step the stale block while eager calls use the other one: the
// advisor's round-5 finding).  Every stream-taking entry point that reads or writes records calls this first; from the first capture
// on, halo launches get no second block and run without halo kitchens.  Engines whose launches can never swap skip the query.
void note_stream(oc_engine *e, hipStream_t s) {
    if (e->state_pinned) return;
#ifndef OC_DIAGNOSTICS
    // (only engines whose planes can start off 64-byte boundaries ever swap -- halo_r_for; the diagnostics build's per-XCD group
    // sizes can make any 2-player engine do it.  The block need not exist yet: the module that brings it may be built after the capture)
    if (e->np_path || (e->n * e->S * kChannels) % 64 == 0) return;
#endif
    hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(s, &cs) != hipSuccess) { (void)hipGetLastError(); return; }
    if (cs != hipStreamCaptureStatusNone) e->state_pinned = true;
}

// The modules that are not part of oc_create's build -- the step entries for fresh (time-major) destinations and the
// K-steps-per-launch rollout entries -- for one geometry: built on first use (or ahead of it by oc_prepare_kernels: hiprtc,
// hipModuleLoadData and the hipDeviceSynchronize of a rebuild have no business inside a stream capture).  A geometry whose build
// failed is remembered and not tried again: the generic ahead-of-time kernel serves it.
bool ensure_side_module(oc_engine *e, JitModule &jm, const Tuning &tu, int which, int waves_per_cu, int fn_first, int fn_last) {
    if (jm.mod && jm.kpw == tu.kpw && jm.gpasses == tu.gpasses) return true;
    if (jm.failed_kpw == tu.kpw && jm.failed_gpasses == tu.gpasses) return false;
    if (jm.mod) { (void)hipDeviceSynchronize(); (void)hipModuleUnload(jm.mod); }
    jm = JitModule();
    jm.failed_kpw = tu.kpw; jm.failed_gpasses = tu.gpasses;             // until the build below succeeds
    std::vector<char> code;
    std::string log;
    hipModule_t m = nullptr;
    if (jit_compile_text(jit_source_single(e, tu, which, waves_per_cu), e->arch, code, log) != OC_OK || hipModuleLoadData(&m, code.data()) != hipSuccess) {
        (void)hipGetLastError();
        return false;
    }
    JitModule j;
    j.mod = m;
    for (int i = fn_first; i <= fn_last; ++i)
        if (hipModuleGetFunction(&j.fn[i], m, kJitNames[i]) != hipSuccess) {
            (void)hipGetLastError();
            (void)hipModuleUnload(m);
            return false;
        }
    j.kpw = tu.kpw; j.gpasses = tu.gpasses;
    if (which == SRC_TWOPTR) { j.xw = xcd_weights(e, tu); j.wg = wg_waves_for(e, tu); }
    if (which == SRC_FRESH) { j.xw = xcd_weights(e, tu); j.wg = wg_waves_for(e, tu); j.halo_r = (!j.xw.sum && !OC_DIAG_ENV("OC_NO_HALO")) ? halo_r_for(e, tu) : 0; }
    jm = j;
    if (which == SRC_FRESH && (j.halo_r || j.xw.sum)) ensure_halo_block(e);
    return true;
}
// (the fused rollout keeps the register budget of the per-step kernel -- 3 waves per SIMD -- not of its own wavefront count: held
// to 128 VGPRs for four waves per SIMD the rollout body measured 7.78 instead of 7.32 us per step)
bool ensure_fresh_module(oc_engine *e, const Tuning &tu) { return ensure_side_module(e, e->jit_fresh, tu, SRC_FRESH, kFreshWavesPerCu, JIT_STEP_I32_V16_NT, JIT_STEP_I64_V16_PL); }
bool ensure_fused_module(oc_engine *e, const Tuning &tu) { return ensure_side_module(e, e->jit_fused, tu, SRC_ROLLOUT, e->waves_per_cu, JIT_ROLLOUT_I32, JIT_ROLLOUT_I64_NT); }
bool ensure_batch_module(oc_engine *e, const Tuning &tu) { return ensure_side_module(e, e->jit_batch, tu, SRC_BATCH, kFreshWavesPerCu, JIT_OBS_BATCH_V16, JIT_OBS_BATCH_V16); }
bool ensure_2p_module(oc_engine *e, const Tuning &tu) { return ensure_side_module(e, e->jit_2p, tu, SRC_TWOPTR, e->waves_per_cu, JIT_STEP_I32_V16_2P, JIT_STEP_I64_V16_2P); }

// A launch of a per-engine (hiprtc) entry point: [p_state, p_tabs, p_actions, p_obs, p_reward, p_done, p_n | StepArgs], see the
// entry points' text in jit_source_single.
hipError_t launch_jit(hipFunction_t fn, const StepArgs &a, unsigned grid, size_t shmem, hipStream_t s, int wg = 1, bool two_ptr = false) {
    if (two_ptr) {                                                    // [seven scalars, p_actions1 | StepArgs]: the SRC_TWOPTR entry points
        struct { uint4 *state; const DevTables *tabs; const void *actions; int8_t *obs; int32_t *reward; int32_t *done; int64_t n; const void *actions1; StepArgs a; } args2 =
            {a.state, a.tabs, a.actions, a.obs, a.reward, a.done, a.n_kitchens, a.actions1, a};
        static_assert(offsetof(decltype(args2), a) == 64, "eight leading scalars, then StepArgs");
        size_t size2 = sizeof(args2);
        void *config2[] = {HIP_LAUNCH_PARAM_BUFFER_POINTER, &args2, HIP_LAUNCH_PARAM_BUFFER_SIZE, &size2, HIP_LAUNCH_PARAM_END};
        return hipModuleLaunchKernel(fn, (grid + wg - 1) / wg, 1, 1, kWave * wg, 1, 1, static_cast<unsigned>(shmem * wg), s, nullptr, config2);
    }
    struct { uint4 *state; const DevTables *tabs; const void *actions; int8_t *obs; int32_t *reward; int32_t *done; int64_t n; StepArgs a; } args =
        {a.state, a.tabs, a.actions, a.obs, a.reward, a.done, a.n_kitchens, a};
    static_assert(offsetof(decltype(args), a) == 56, "seven leading scalars, then StepArgs");
    size_t size = sizeof(args);
    void *config[] = {HIP_LAUNCH_PARAM_BUFFER_POINTER, &args, HIP_LAUNCH_PARAM_BUFFER_SIZE, &size, HIP_LAUNCH_PARAM_END};
    // (wg wavefronts per workgroup: `grid` counts wavefronts)
    return hipModuleLaunchKernel(fn, (grid + wg - 1) / wg, 1, 1, kWave * wg, 1, 1, static_cast<unsigned>(shmem * wg), s, nullptr, config);
}

// ... and the swap behind such a launch.  (Diagnostics build: the folded env step keeps a device-resident copy of its step arguments,
// state pointer included -- oc_internal_fold_workspace -- which follows the swap, stream-ordered.)
hipError_t swap_state_blocks(oc_engine *e, hipStream_t s) {
    std::swap(e->d_state, e->d_state_alt);
#ifdef OC_DIAGNOSTICS
    if (e->d_fold_args)
        return hipMemcpyAsync(reinterpret_cast<char *>(e->d_fold_args) + offsetof(StepArgs, state), &e->d_state, sizeof(e->d_state), hipMemcpyHostToDevice, s);
#endif
    (void)s;
    return hipSuccess;
}

// in-place planes larger than this are stored like fresh destinations (launch)
constexpr int64_t kStreamInPlaceBytes = 320ll << 20;

template <bool STEP, bool ACT64>
int launch(oc_engine *e, const StepArgs &a_in, hipStream_t s, bool fresh_geom = false) {
    StepArgs a = a_in;
    if (a.n_kitchens == 0) return OC_OK;
    const bool vec16 = wide_stores();
    // persistent waves: at most waves_per_cu per CU, each walking its groups in a grid-stride loop
    const int wpc = fresh_geom ? kFreshWavesPerCu : e->waves_per_cu;
    const unsigned grid = static_cast<unsigned>(min(static_cast<int64_t>(a.n_groups), static_cast<int64_t>(wpc) * launch_cus(e)));
    // (the per-engine entry points with per-XCD group sizes count their groups differently: xcd_weights)
    auto grid_of = [&](const JitModule &m) {
        if (!m.xw.sum) return grid;
        const int64_t g8 = min(xcd_groups(m.xw, a.n_kitchens), static_cast<int64_t>(wpc) * launch_cus(e));
        return static_cast<unsigned>(g8 >= 8 ? g8 - g8 % 8 : g8);
    };
    const size_t shmem = lds_bytes(e, a.kpw, a.gpasses);
    // per-engine build when there is one for the current tuning (diagnostic traces: generic kernel)
    if (!fresh_geom && vec16 && e->jit.mod && e->jit.kpw == a.kpw && e->jit.gpasses == a.gpasses && (!a.trace || OC_DIAG_ENV("OC_JIT_TRACE"))) {
        // a destination that differs from the previous step's is a trajectory slot, not an in-place buffer:
        // stream it past the caches (see store16).  So is an in-place buffer that the Infinity Cache (256 MB) cannot hold anyway:
        // write-through stores that allocate there only evict each other -- in place, `sc1` / `sc1 nt`, us per launch
        // (profiles/r04_ab_bign.log): cramped_room 131 072 kitchens (105 MB of planes) 19.5 / 20.4, 262 144 (210 MB) 38.7 / 38.2,
        // 524 288 (419 MB) 78.8 / 76.5, 10^6 (800 MB) 169 / 146; asymmetric_advantages 131 072 (236 MB) 42.3 / 43.2, 262 144 (472 MB) 111 / 91
        const bool beyond_cache = 2 * a.obs_player_stride > kStreamInPlaceBytes;
        const bool nt = STEP && (a.obs != e->last_obs || beyond_cache);
        const bool pl = nt && e->planes_read_next;
        const int idx = STEP ? (ACT64 ? (pl ? JIT_STEP_I64_V16_PL : nt ? JIT_STEP_I64_V16_NT : JIT_STEP_I64_V16)
                                      : (pl ? JIT_STEP_I32_V16_PL : nt ? JIT_STEP_I32_V16_NT : JIT_STEP_I32_V16))
                             : JIT_OBS_V16;
        if (STEP && e->jit.xw.sum) {                         // (diagnostics build only: per-XCD group sizes have halo kitchens)
            ensure_halo_block(e);
            if (a.state != e->d_state || !(a.state_out = halo_state_out(e, s))) return fail(OC_ERR_UNSUPPORTED, "per-XCD group sizes: no second state block for this launch");
        }
        OC_HIP(launch_jit(e->jit.fn[idx], a, grid_of(e->jit), shmem, s, idx == JIT_OBS_BATCH_V16 ? 1 : e->jit.wg));
        if (a.state_out) OC_HIP(swap_state_blocks(e, s));
        if (STEP) e->last_obs = a.obs;
        return OC_OK;
    }
    // a step into a fresh destination with the geometry kept for those (step_impl chose it): its own module, built here once
    if (STEP && fresh_geom && vec16 && e->jit.mod && (!a.trace || OC_DIAG_ENV("OC_JIT_TRACE"))) {
        if (ensure_fresh_module(e, fresh_tuning(e))) {
            const size_t shmem_f = e->jit_fresh.halo_r ? lds_bytes(e, a.kpw + 1, a.gpasses) + kHaloCarryBytes : shmem;
            if ((e->jit_fresh.halo_r && !e->planes_read_next) || e->jit_fresh.xw.sum) {
                a.state_out = a.state == e->d_state ? halo_state_out(e, s) : nullptr;
                if (!a.state_out && e->jit_fresh.xw.sum) return fail(OC_ERR_UNSUPPORTED, "per-XCD group sizes: no second state block for this launch");
            }
            OC_HIP(launch_jit(e->jit_fresh.fn[e->planes_read_next ? (ACT64 ? JIT_STEP_I64_V16_PL : JIT_STEP_I32_V16_PL)
                                                                  : (ACT64 ? JIT_STEP_I64_V16_NT : JIT_STEP_I32_V16_NT)], a, grid_of(e->jit_fresh), shmem_f, s, e->jit_fresh.wg));
            if (a.state_out) OC_HIP(swap_state_blocks(e, s));
            e->last_obs = a.obs;
            return OC_OK;
        }
    }
    if (vec16) launch_v<STEP, ACT64, true>(a, grid, shmem, s);
    else launch_v<STEP, ACT64, false>(a, grid, shmem, s);
    OC_HIP(hipGetLastError());
    return OC_OK;
}

template <bool ACT64, bool VEC16, int QN>
void launch_rollout_q(const StepArgs &a, unsigned grid, size_t shmem, hipStream_t s) {
    hipLaunchKernelGGL((oc_rollout_kernel<ACT64, VEC16, QN>), dim3(grid), dim3(kWave), shmem, s, a);
}

template <bool ACT64, bool VEC16>
void launch_rollout_v(const StepArgs &a, unsigned grid, size_t shmem, hipStream_t s) {
    switch (qn_for(a.kpw, a.recq)) {
    case 2: launch_rollout_q<ACT64, VEC16, 2>(a, grid, shmem, s); break;
    case 3: launch_rollout_q<ACT64, VEC16, 3>(a, grid, shmem, s); break;
    case 4: launch_rollout_q<ACT64, VEC16, 4>(a, grid, shmem, s); break;
    default: launch_rollout_q<ACT64, VEC16, kMaxQ>(a, grid, shmem, s); break;
    }
}

// One launch for a whole rollout: every wave keeps its kitchens' state in LDS across the steps.
int launch_fused(oc_engine *e, const StepArgs &a, bool act64, hipStream_t s) {
    if (a.n_kitchens == 0 || a.n_steps == 0) return OC_OK;
    const bool vec16 = wide_stores();
    const size_t shmem = lds_bytes(e, a.kpw, a.gpasses);
    // A wavefront runs ALL steps of a group before it takes its next one, so a wavefront with two groups takes twice as long
    // as one with one: use every wavefront the CUs can hold (LDS, and 4 per SIMD by registers) rather than the per-step
    // kernel's persistent count -- 65 536 kitchens in groups of 16 are 4096 groups on 16 x 256 wavefronts, one each
    // (8.6 -> 7.7 us per step against 12 per CU).
    const int fused_wpc = e->tuned_by_user ? e->waves_per_cu
                                           : static_cast<int>(std::max<size_t>(8, std::min<size_t>(16, 160 * 1024 / shmem)));
    const unsigned grid = static_cast<unsigned>(min(static_cast<int64_t>(a.n_groups), static_cast<int64_t>(fused_wpc) * launch_cus(e)));
    // the specialised build for this geometry: the rollout-only module, built on the first rollout
    const JitModule *mod = nullptr;
    if (e->jit.mod && vec16 && !a.trace) {
        if (ensure_fused_module(e, Tuning{a.kpw, a.gpasses, a.kpp})) mod = &e->jit_fused;
    }
    if (mod && vec16 && !a.trace) {
        const bool nt = a.obs_step_stride != 0;          // fresh slot per step: stream past the caches
        const int idx = act64 ? (nt ? JIT_ROLLOUT_I64_NT : JIT_ROLLOUT_I64) : (nt ? JIT_ROLLOUT_I32_NT : JIT_ROLLOUT_I32);
        OC_HIP(launch_jit(mod->fn[idx], a, grid, shmem, s));
        e->last_obs = nullptr;
        return OC_OK;
    }
    if (act64) { if (vec16) launch_rollout_v<true, true>(a, grid, shmem, s); else launch_rollout_v<true, false>(a, grid, shmem, s); }
    else { if (vec16) launch_rollout_v<false, true>(a, grid, shmem, s); else launch_rollout_v<false, false>(a, grid, shmem, s); }
    OC_HIP(hipGetLastError());
    e->last_obs = nullptr;
    return OC_OK;
}

// Wait for an event the way a latency-sensitive caller does: poll it for a while before handing the thread to the blocking
// wait (whose wake-up costs tens of microseconds: a timed rollout of 20 steps is 235 us of kernels).
hipError_t wait_event(hipEvent_t ev) {
    for (int i = 0; i < 200000; ++i) {
        const hipError_t q = hipEventQuery(ev);
        if (q == hipSuccess) return hipSuccess;
        if (q != hipErrorNotReady) { (void)hipGetLastError(); return q; }
    }
    (void)hipGetLastError();                                 // (hipErrorNotReady is sticky in hipGetLastError)
    return hipEventSynchronize(ev);
}

int check_engine(const oc_engine *e) {
    if (!e) return fail(OC_ERR_INVALID_ARG, "engine handle is NULL");
    return OC_OK;
}

// Every entry point that enqueues work runs with the engine's GPU current and hands the caller's device back
// on return (two engines on different GPUs in one process, torch.cuda.set_device between calls).
#define OC_ON_ENGINE_DEVICE(e)                                                                        \
    const OcDeviceScope on_device__((e)->device);                                                     \
    if (!on_device__.ok) return fail(OC_ERR_HIP, "cannot make device %d current", (e)->device)

int np_step(oc_engine *e, const void *actions, int action_dtype, int8_t *obs, int32_t *reward, int32_t *done, void *records, hipStream_t s);
int np_encode(oc_engine *e, const uint32_t *state, int64_t n, int8_t *obs, int64_t obs_player_stride, hipStream_t s, void *records = nullptr);

// d_records (may be NULL): where the post-step state records of all kitchens also go, [N][record bytes], 16-byte aligned (checked
// by the callers) -- the trajectory's record slot, written by the launch that computed the records
int step_impl(oc_engine *e, const void *d_actions, int action_dtype, int8_t *d_obs, int32_t *d_reward,
              int32_t *d_done, void *d_records, hipStream_t s) {
    if (e->np_path) return np_step(e, d_actions, action_dtype, d_obs, d_reward, d_done, d_records, s);
    // a destination that differs from the previous step's is a trajectory slot: the geometry kept for those (fresh_tuning)
    const bool fresh = d_obs != e->last_obs && e->last_obs != nullptr && has_fresh_geometry(e);
    StepArgs a = fresh ? make_args(e, fresh_tuning(e), e->d_state, e->n, d_actions, d_obs, d_reward, d_done)
                       : make_args(e, e->d_state, e->n, d_actions, d_obs, d_reward, d_done);
    a.rec_out = static_cast<uint4 *>(d_records);
    return action_dtype == OC_ACT_I64 ? launch<true, true>(e, a, s, fresh) : launch<true, false>(e, a, s, fresh);
}


template <bool VEC16>
void launch_observe_batch_generic(const StepArgs &a, unsigned grid, size_t shmem, hipStream_t s) {
    switch (qn_for(a.kpw, a.recq)) {
    case 2: hipLaunchKernelGGL((oc_observe_batch_kernel<VEC16, 2>), dim3(grid), dim3(kWave), shmem, s, a); break;
    case 3: hipLaunchKernelGGL((oc_observe_batch_kernel<VEC16, 3>), dim3(grid), dim3(kWave), shmem, s, a); break;
    case 4: hipLaunchKernelGGL((oc_observe_batch_kernel<VEC16, 4>), dim3(grid), dim3(kWave), shmem, s, a); break;
    default: hipLaunchKernelGGL((oc_observe_batch_kernel<VEC16, kMaxQ>), dim3(grid), dim3(kWave), shmem, s, a); break;
    }
}

// `a` describes ONE item (n records -> two viewer planes); `items` of them, strides already set.
// A whole trajectory is a large batch whatever the engine's own kitchen count: an engine whose launch geometry was chosen for a
// small batch (one GPU's share of config 4: 8192 kitchens, 8 per group) re-featurises T x n kitchens with the geometry of fresh
// destinations instead -- 16 per group, four passes per flush, eight wavefronts per CU, from a module of its own
// (tools/exp_encode_trajectory.py: 0.92 -> 0.65 ms = 3.2 -> 4.5 TB/s written at 8192 asymmetric_advantages kitchens x 200 steps).
int launch_observe_batch(oc_engine *e, StepArgs a, int64_t items, hipStream_t s) {
    if (a.n_kitchens == 0 || items == 0) return OC_OK;
    const bool vec16 = wide_stores();
    int wpc = e->waves_per_cu;
    const JitModule *mod = (vec16 && e->jit.mod && e->jit.kpw == a.kpw && e->jit.gpasses == a.gpasses && !a.trace) ? &e->jit : nullptr;
    // (an engine that already runs 16 per group keeps its own geometry: 5.17 ms against 5.39 at 65 536 kitchens)
    if (mod && !e->tuned_by_user && a.kpw < 16 && 16 * e->recq <= kMaxQ * kWave && (a.n_kitchens + 15) / 16 * items >= 3072) {
        const Tuning big{16, 4, kpp_for(e->S, 4)};
        if (ensure_batch_module(e, big)) {
            const StepArgs b = make_args(e, big, a.state, a.n_kitchens, nullptr, a.obs, nullptr, nullptr);
            const int64_t ops = a.obs_player_stride, sbs = a.state_batch_stride, obs_bs = a.obs_batch_stride;
            a = b;
            a.obs_player_stride = ops; a.state_batch_stride = sbs; a.obs_batch_stride = obs_bs;
            mod = &e->jit_batch;
            wpc = kFreshWavesPerCu;
        }
    }
    a.batch_groups = a.n_groups;
    if (a.batch_groups * items > 0x7fffffff) return fail(OC_ERR_INVALID_ARG, "oc_encode_trajectory: too many groups for one launch");
    a.n_groups = static_cast<int32_t>(a.batch_groups * items);
    const unsigned grid = static_cast<unsigned>(min(static_cast<int64_t>(a.n_groups), static_cast<int64_t>(wpc) * launch_cus(e)));
    const size_t shmem = lds_bytes(e, a.kpw, a.gpasses);
    if (mod) {
        OC_HIP(launch_jit(mod->fn[JIT_OBS_BATCH_V16], a, grid, shmem, s));
        return OC_OK;
    }
    if (vec16) launch_observe_batch_generic<true>(a, grid, shmem, s);
    else launch_observe_batch_generic<false>(a, grid, shmem, s);
    OC_HIP(hipGetLastError());
    return OC_OK;
}

// ---- kitchens with 1, 3 or 4 players: the group kernel of oc_np_kernels.h
oc_np::NpArgs np_args(const oc_engine *e, uint32_t *state, int64_t n, const void *actions, int act64, int8_t *obs, int64_t obs_player_stride,
                      int32_t *reward, int32_t *done) {
    oc_np::NpArgs a;
    a.state = state;
    a.tabs = e->d_tabs;                                // the table image: tile map, terrain, recipe tables (its head is copied to LDS)
    a.actions = actions; a.act64 = act64;
    a.obs = obs; a.obs_player_stride = obs_player_stride;
    a.reward = reward; a.done = done;
    a.n = n;
    a.W = e->params.width; a.H = e->params.height; a.S = e->S; a.P = e->P; a.C = 5 * e->P + 10; a.recd = e->recd;
    a.horizon = e->params.horizon; a.placement_rew = e->params.placement_in_pot_rew; a.soup_rew = e->params.soup_pickup_rew;
    for (int i = 0; i < 4; ++i) a.start_pp[i] = e->start_pp[i];
    a.rec_out = nullptr;
    a.items = 1; a.state_item_stride = 0; a.obs_item_stride = 0;
    a.n_steps = 1; a.tape_steps = 1; a.obs_step_stride = 0; a.reward_step_stride = 0; a.done_step_stride = 0; a.rec_step_stride = 0;
    a.no_pipeline = OC_DIAG_ENV("OC_NP_NOPIPE") ? atoi(OC_DIAG_ENV("OC_NP_NOPIPE")) : 0;
    return a;
}

// Launch geometry of the N-player kernel: 16 kitchens per group (K x P <= 64 poke lanes), fewer on batches that would leave CUs
// without a wavefront; G passes per flush; as many persistent wavefronts per CU as LDS holds, at most eight.
oc_np::NpGeom np_geometry(const oc_engine *e, int64_t n) {       // n: kitchens of the launch (all items of a batched featurisation)
    if (e->tuned_by_user) return oc_np::NpGeom{e->kpw, e->gpasses};
    // (profiles/r05_np_sweep.log, us per step at 65 536 kitchens: one player 32 / 4 12.8 against 14.7 with 16 / 2; three players
    // 16 / 3 59.6 against 61.4; four players 16 / 2 best; 8192 kitchens: groups of 4 on sixteen wavefronts per CU 16.4 against 25.2)
    int K = e->P == 1 ? 32 : 16;
    while (K > 1 && K * e->recq > 256) K /= 2;                      // the prefetch window: four 16-byte chunks per lane
    while (K > 4 && (n + K - 1) / K < 8ll * launch_cus(e)) K /= 2;  // small batches: a group for every wavefront the CUs hold
    return oc_np::NpGeom{K, e->P == 1 ? 4 : e->P == 3 ? 3 : 2};
}

template <bool STEP, int SM, bool FUSED = false, bool BATCH = false>
int np_launch_sm(oc_engine *e, const oc_np::NpArgs &a, unsigned grid, size_t shmem, hipStream_t s) {
    switch (e->P) {
    case 1: hipLaunchKernelGGL((oc_np::np_group_kernel<1, STEP, SM, FUSED, BATCH>), dim3(grid), dim3(kWave), shmem, s, a); break;
    case 3: hipLaunchKernelGGL((oc_np::np_group_kernel<3, STEP, SM, FUSED, BATCH>), dim3(grid), dim3(kWave), shmem, s, a); break;
    case 4: hipLaunchKernelGGL((oc_np::np_group_kernel<4, STEP, SM, FUSED, BATCH>), dim3(grid), dim3(kWave), shmem, s, a); break;
    default: return fail(OC_ERR_UNSUPPORTED, "no N-player kernel for %d players", e->P);
    }
    OC_HIP(hipGetLastError());
    return OC_OK;
}

template <bool STEP>
int np_launch(oc_engine *e, oc_np::NpArgs a, hipStream_t s) {
    if (a.n == 0) return OC_OK;
    const oc_np::NpGeom g = np_geometry(e, a.n * a.items);
    a.K = g.K; a.G = g.G;
    a.inv_S = 1.0f / static_cast<float>(e->S); a.inv_H = 1.0f / static_cast<float>(e->params.height);
    a.inv_W = 1.0f / static_cast<float>(e->params.width); a.inv_recq = 1.0f / static_cast<float>(e->recq);
    const size_t shmem = oc_np::np_lds_bytes(e->S, e->P, e->recd, g);
    if (shmem > 64 * 1024) return fail(OC_ERR_UNSUPPORTED, "%d-player kitchens of %d tiles need %zu bytes of LDS per wavefront", e->P, e->S, shmem);
    const int wpc = static_cast<int>(std::max<size_t>(1, std::min<size_t>(e->tuned_by_user ? e->waves_per_cu : (g.K < 16 ? 16 : 8), 160 * 1024 / shmem)));
    const int64_t groups = (a.n + g.K - 1) / g.K * a.items;
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(groups, static_cast<int64_t>(wpc) * launch_cus(e)));
    // plane stores: write-through while the planes of a launch fit the 256 MB Infinity Cache (the next launch of a rollout overwrites
    // them there), plain beyond it (profiles/r05_np_sweep.log: 4 x 65 536 kitchens, 385 MB of planes: 83 us plain, 107 sc1, 109 sc1 nt;
    // 4 x 8192: 17.8 plain, 16.4 sc1)
    // What counts is everything the launch (or the run of launches) writes before it comes back to the same bytes: a K-steps launch
    // with a slot per step writes n_steps x the planes, and a step whose destination differs from the previous step's is a
    // time-major slot of a trajectory far larger than the cache -- both are stored plainly (the rule looked at
    // one step's planes only).
    const int64_t planes = static_cast<int64_t>(e->P) * a.obs_player_stride;
    const int64_t footprint = (STEP && a.n_steps > 1 && a.obs_step_stride > 0) ? planes + a.obs_step_stride * (static_cast<int64_t>(a.n_steps) - 1) : planes;
    const bool fresh_slot = STEP && a.n_steps <= 1 && e->last_obs != nullptr && a.obs != e->last_obs;
    int sm = (footprint <= (200ll << 20) && !fresh_slot) ? SM_SC1 : SM_PLAIN;
    if (STEP) e->last_obs = a.n_steps <= 1 ? a.obs : nullptr;
    if (const char *v = OC_DIAG_ENV("OC_NP_SM")) sm = atoi(v);
#ifdef OC_DIAGNOSTICS
    if (sm == SM_SC1_NT) return np_launch_sm<STEP, SM_SC1_NT>(e, a, grid, shmem, s);
    if (sm == SM_NT) return np_launch_sm<STEP, SM_NT>(e, a, grid, shmem, s);
#endif
    if (!STEP && a.items > 1) {                              // a whole trajectory: the build whose groups run over all items (fresh planes)
        if (groups > 0x7fffffff) return fail(OC_ERR_INVALID_ARG, "oc_encode_trajectory: too many groups for one launch");
        return np_launch_sm<false, SM_PLAIN, false, !STEP>(e, a, grid, shmem, s);
    }
    if (STEP && a.n_steps > 1) {                             // K steps per launch: the build with the step loop
        if (sm == SM_SC1) return np_launch_sm<STEP, SM_SC1, STEP>(e, a, grid, shmem, s);
        return np_launch_sm<STEP, SM_PLAIN, STEP>(e, a, grid, shmem, s);
    }
    if (sm == SM_SC1) return np_launch_sm<STEP, SM_SC1>(e, a, grid, shmem, s);
    return np_launch_sm<STEP, SM_PLAIN>(e, a, grid, shmem, s);
}

int np_encode(oc_engine *e, const uint32_t *state, int64_t n, int8_t *obs, int64_t obs_player_stride, hipStream_t s, void *records) {
    oc_np::NpArgs a = np_args(e, const_cast<uint32_t *>(state), n, nullptr, 0, obs, obs_player_stride, nullptr, nullptr);
    a.rec_out = static_cast<uint32_t *>(records);
    return np_launch<false>(e, a, s);
}

// ONE launch per step: transition, encoding of every viewer, reward, done and -- records != NULL -- the trajectory's record slot
int np_step(oc_engine *e, const void *actions, int action_dtype, int8_t *obs, int32_t *reward, int32_t *done, void *records, hipStream_t s) {
    oc_np::NpArgs a = np_args(e, reinterpret_cast<uint32_t *>(e->d_state), e->n, actions, action_dtype == OC_ACT_I64 ? 1 : 0, obs,
                              e->n * e->S * (5 * e->P + 10), reward, done);
    a.rec_out = static_cast<uint32_t *>(records);
    return np_launch<true>(e, a, s);
}

#define OC_TWO_PLAYER_ONLY(e, who)                                                                                      \
    if ((e)->np_path) return fail(OC_ERR_UNSUPPORTED, "%s: 2-player kitchens only (this engine has %d players)", who, (e)->P)

}  // namespace

// ---- several engines stepped by one launch ---------------------------------------------------------------
struct oc_group {
    std::vector<oc_engine *> engines;
    std::vector<Tuning> tunings;
    std::vector<int> layout_of_seg, blocks;
    int device, waves_per_cu, num_cus;
    hipModule_t mod;
    hipFunction_t fn[GJIT_NFUNC];
    size_t shmem;
    const int8_t *last_obs0;
    char status[256];
};

namespace {

void group_unload(oc_group *g) {
    if (g->mod) (void)hipModuleUnload(g->mod);
    g->mod = nullptr;
}

// Launch geometry of a group.  A launch is as long as its slowest wavefront, so the persistent wavefronts of the chip
// (waves_per_cu x CUs) must end up with equal amounts of tiles whatever mix of grids they serve:
//   * small joint batches (every wavefront can get exactly one group): the smallest per-wavefront tile budget tau for
//     which kpw_i = 4 * floor(tau / (4 S_i)) kitchens per group leave no more groups than wavefronts -- one group per
//     wavefront, no wavefront with two (5 x 8192 kitchens on 12 x 256 wavefronts -> 24/8/20/20/12 kitchens
//     per group, <= 500 tiles each);
//   * large batches: the single-engine defaults, wavefronts shared out in proportion to the engines' tiles.
int group_plan(oc_group *g, const int32_t *kpw_override, int passes, int waves_per_cu) {
    const int n = static_cast<int>(g->engines.size());
    if (waves_per_cu) g->waves_per_cu = waves_per_cu;
    const int64_t slots = static_cast<int64_t>(g->waves_per_cu) * g->num_cus;
    double total = 0;
    for (const oc_engine *e : g->engines) total += static_cast<double>(e->n) * e->S;
    auto kpw_cap = [&](const oc_engine *e) {
        int cap = 64;
        while (cap > 4 && cap * e->recq > kMaxQ * kWave) cap -= 4;
        return cap;
    };
    auto groups_of = [&](const oc_engine *e, int kpw) { return (e->n + kpw - 1) / kpw; };
    std::vector<int> kpw(n, 0);
    bool one_group_each = false;
    for (int tau = 64; tau <= 64 * 255 && !one_group_each; tau += 4) {
        int64_t need = 0;
        for (int i = 0; i < n; ++i) {
            const oc_engine *e = g->engines[i];
            const int k = std::min(kpw_cap(e), tau / (4 * e->S) * 4);
            if (k < 4) { need = slots + 1; break; }
            kpw[i] = k;
            need += groups_of(e, k);
        }
        one_group_each = need <= slots;
    }
    if (!one_group_each)
        for (int i = 0; i < n; ++i) kpw[i] = std::min(kpw_cap(g->engines[i]), 16);       // the single-engine default for large batches
    // The small grids (at most 32 tiles) flush full groups in one batch (oc_step_body.h) and like group sizes of 16 or 32 kitchens
    // better than what equal tiles per wavefront gives them: config 3's 24 / 8 / 20 / 20 / 12 -> 32 / 8 / 16 / 16 / 12 measured
    // 12.59 against 12.90 us per joint step.
    if (one_group_each)
        for (int i = 0; i < n; ++i) {
            const oc_engine *e = g->engines[i];
            if (e->S > 32 || kpw[i] < 16) continue;
            const int snapped = kpw[i] >= 24 && 32 * e->recq <= kMaxQ * kWave && (32 * e->S) % kWave == 0 ? 32 : 16;
            kpw[i] = snapped;
        }
    g->tunings.resize(n);
    g->blocks.assign(n, 1);
    size_t lds = 0;
    for (int i = 0; i < n; ++i) {
        const oc_engine *e = g->engines[i];
        if (kpw_override && kpw_override[i]) kpw[i] = kpw_override[i];
        if (kpw[i] < 1 || kpw[i] > 64 || (kpw[i] * e->S * 5) % 4 || kpw[i] * e->recq > kMaxQ * kWave)
            return fail(OC_ERR_INVALID_ARG, "oc_group_set_tuning: kitchens_per_wave %d is not usable for engine %d (1..64, kitchens*tiles a multiple of 4, "
                        "at most %d B of records per group)", kpw[i], i, kMaxQ * kWave * 16);
        int gp = passes ? passes : 2;                                 // 2 passes per flush, 12 wavefronts per CU: 12.73 vs 13.14 us on config 3 with 4 / 8
        if (gp < 1 || gp > 8) return fail(OC_ERR_INVALID_ARG, "oc_group_set_tuning: passes_per_flush must be in 1..8");
        while (gp > 1 && lds_bytes(e, kpw[i], gp) * g->waves_per_cu > 160 * 1024) --gp;
        g->tunings[i] = Tuning{kpw[i], gp, kpp_for(e->S, gp)};
        lds = std::max(lds, lds_bytes(e, kpw[i], gp));
    }
    if (lds > 64 * 1024) return fail(OC_ERR_INVALID_ARG, "oc_group: %zu B of LDS per wavefront exceeds 64 KiB", lds);
    g->shmem = lds;
    // wavefronts per engine: all its groups if everything fits, else in proportion to its tiles (at least 1, at most its
    // groups); what is left over goes to whoever has the most groups per wavefront
    std::vector<int64_t> groups(n);
    int64_t used = 0, all = 0;
    for (int i = 0; i < n; ++i) { groups[i] = groups_of(g->engines[i], kpw[i]); all += groups[i]; }
    for (int i = 0; i < n; ++i) {
        const oc_engine *e = g->engines[i];
        const int64_t share = static_cast<int64_t>(static_cast<double>(slots) * (static_cast<double>(e->n) * e->S / total));
        g->blocks[i] = static_cast<int>(all <= slots ? groups[i] : std::max<int64_t>(1, std::min<int64_t>(groups[i], share)));
        used += g->blocks[i];
    }
    while (used < slots) {
        int best = -1;
        double worst = 1.0;
        for (int i = 0; i < n; ++i)
            if (g->blocks[i] < groups[i] && static_cast<double>(groups[i]) / g->blocks[i] > worst) {
                worst = static_cast<double>(groups[i]) / g->blocks[i];
                best = i;
            }
        if (best < 0) break;
        ++g->blocks[best];
        ++used;
    }
    return OC_OK;
}

void group_build(oc_group *g) {
    group_unload(g);
    if (jit_disabled(g->engines[0], g->status, sizeof(g->status))) return;
    std::vector<const oc_engine *> es(g->engines.begin(), g->engines.end());
    std::vector<char> code;
    std::string log;
    const char *from = "";
    const std::string text = jit_source_group(es, g->tunings, (g->waves_per_cu + 3) / 4, g->layout_of_seg);
    if (jit_compile_text(text, g->engines[0]->arch, code, log, &from) != OC_OK) {
        snprintf(g->status, sizeof(g->status), "hiprtc: %.220s", log.c_str());
        return;
    }
    hipModule_t mod = nullptr;
    if (hipModuleLoadData(&mod, code.data()) != hipSuccess) {
        (void)hipGetLastError();
        snprintf(g->status, sizeof(g->status), "hipModuleLoadData failed");
        return;
    }
    for (int i = 0; i < GJIT_NFUNC; ++i)
        if (hipModuleGetFunction(&g->fn[i], mod, kGroupJitNames[i]) != hipSuccess) {
            (void)hipGetLastError();
            (void)hipModuleUnload(mod);
            snprintf(g->status, sizeof(g->status), "entry point %s missing", kGroupJitNames[i]);
            return;
        }
    g->mod = mod;
    int n_layouts = 0;
    for (int l : g->layout_of_seg) n_layouts = std::max(n_layouts, l + 1);
    int off = snprintf(g->status, sizeof(g->status), "one launch, %d engines, %d specialised bodies for %s (%s); kpw/blocks", static_cast<int>(g->engines.size()),
                       n_layouts, g->engines[0]->arch, from);
    for (size_t i = 0; i < g->engines.size() && off < static_cast<int>(sizeof(g->status)) - 16; ++i)
        off += snprintf(g->status + off, sizeof(g->status) - off, " %d/%d", g->tunings[i].kpw, g->blocks[i]);
}

int group_launch(oc_group *g, int fn_index, GroupArgs &m, hipStream_t s) {
    unsigned grid = 0;
    m.n_segs = static_cast<int32_t>(g->engines.size());
    for (int i = 0; i <= kMaxSegments; ++i) {              // segment i owns blocks [first_block[i], first_block[i + 1])
        m.first_block[i] = static_cast<int32_t>(grid);
        if (i < kMaxSegments) m.seg_layout[i] = i < m.n_segs ? g->layout_of_seg[i] : -1;
        if (i < m.n_segs) grid += static_cast<unsigned>(g->blocks[i]);
    }
    // [segment count, first blocks 1..8, layout indices (4 bits each), pad | GroupArgs]: see the entry points' text in jit_source_group
    struct { int32_t n_segs, f[8]; uint32_t layouts; int32_t pad[2]; GroupArgs m; } args;
    static_assert(offsetof(decltype(args), m) == 48, "twelve leading dwords, then GroupArgs");
    args.n_segs = m.n_segs;
    args.layouts = 0;
    for (int i = 0; i < kMaxSegments; ++i) {
        args.f[i] = m.first_block[i + 1];
        if (i < m.n_segs) args.layouts |= static_cast<uint32_t>(m.seg_layout[i] & 15) << (4 * i);
    }
    args.pad[0] = args.pad[1] = 0;
    args.m = m;
    size_t size = sizeof(args);
    void *config[] = {HIP_LAUNCH_PARAM_BUFFER_POINTER, &args, HIP_LAUNCH_PARAM_BUFFER_SIZE, &size, HIP_LAUNCH_PARAM_END};
    OC_HIP(hipModuleLaunchKernel(g->fn[fn_index], grid, 1, 1, kWave, 1, 1, static_cast<unsigned>(g->shmem), s, nullptr, config));
    return OC_OK;
}

int check_group(const oc_group *g) {
    if (!g) return fail(OC_ERR_INVALID_ARG, "group handle is NULL");
    return OC_OK;
}

#define OC_ON_GROUP_DEVICE(g)                                                                         \
    const OcDeviceScope on_device__((g)->device);                                                     \
    if (!on_device__.ok) return fail(OC_ERR_HIP, "cannot make device %d current", (g)->device)

}  // namespace

int oc_internal_set_cu_budget(oc_engine *e, int cus) {
    if (int rc = check_engine(e)) return rc;
    if (cus < 0) return fail(OC_ERR_INVALID_ARG, "set_cu_budget: negative CU count");
    e->cu_budget = cus;
    return OC_OK;
}

oc_engine *oc_internal_group_engine(oc_group *g, int i) {
    return (g && i >= 0 && i < static_cast<int>(g->engines.size())) ? g->engines[i] : nullptr;
}

#ifdef OC_DIAGNOSTICS
int oc_internal_fold_args(oc_engine *e, const void *d_actions, int8_t *d_obs, int32_t *d_reward, int32_t *d_done, oc_dev::StepArgs *out,
                          size_t *lds_need) {
    if (!e || !out) return fail(OC_ERR_INVALID_ARG, "fold: NULL argument");
    if (e->np_path) return fail(OC_ERR_UNSUPPORTED, "fold: 2-player kitchens only");
    if (kFoldKpw * e->recq > kFoldQN * kWave || (kFoldKpw * e->S * 5) % 4)
        return fail(OC_ERR_UNSUPPORTED, "fold: %d-byte records exceed the fold's prefetch window", e->recq * 16);
    const Tuning tu{kFoldKpw, kFoldPasses, 0};
    *out = make_args(e, tu, e->d_state, e->n, d_actions, d_obs, d_reward, d_done);
    if (!OC_DIAG_ENV("OC_FOLD_TRACE")) out->trace = nullptr;              // diagnostics: the phase stamps of the folded body (oc_debug_trace first)
    out->ablate = 0;
    if (lds_need) *lds_need = lds_bytes(e, tu.kpw, tu.gpasses);
    return OC_OK;
}

int oc_internal_fold_workspace(oc_engine *e, int32_t **d_count, int32_t **d_expected, int32_t *n_groups, const oc_dev::StepArgs **d_args_template) {
    if (!e || !d_count || !d_expected || !n_groups || !d_args_template) return fail(OC_ERR_INVALID_ARG, "fold: NULL argument");
    const int64_t g = (e->n + kFoldKitchens - 1) / kFoldKitchens;
    if (g > 0x3fffffff) return fail(OC_ERR_UNSUPPORTED, "fold: too many kitchens");
    if (!e->d_fold_ws) {
        OC_ON_ENGINE_DEVICE(e);
        StepArgs tmpl;
        if (int rc = oc_internal_fold_args(e, nullptr, nullptr, nullptr, nullptr, &tmpl, nullptr)) return rc;
        OC_HIP(hipMalloc(reinterpret_cast<void **>(&e->d_fold_args), sizeof(StepArgs)));
        OC_HIP(hipMemcpy(e->d_fold_args, &tmpl, sizeof(StepArgs), hipMemcpyHostToDevice));
        OC_HIP(hipMalloc(reinterpret_cast<void **>(&e->d_fold_ws), static_cast<size_t>(2 * g) * sizeof(int32_t)));
        OC_HIP(hipMemset(e->d_fold_ws, 0, static_cast<size_t>(2 * g) * sizeof(int32_t)));
    }
    *d_count = e->d_fold_ws;
    *d_expected = e->d_fold_ws + g;
    *n_groups = static_cast<int32_t>(g);
    *d_args_template = e->d_fold_args;
    return OC_OK;
}
#endif  // OC_DIAGNOSTICS

void oc_internal_note_destination(oc_engine *e, const int8_t *d_obs) { if (e) e->last_obs = d_obs; }
void oc_internal_planes_read_next(oc_engine *e, int on) {
    static const bool disabled = [] { const char *v = OC_DIAG_ENV("OC_PLAIN_FRESH"); return v && v[0] == '0'; }();   // diagnostics: OC_PLAIN_FRESH=0 keeps the streaming stores
    if (e) e->planes_read_next = on != 0 && !disabled;
}

extern "C" {

const char *oc_last_error(void) { return g_err; }
int oc_abi_version(void) { return OC_ABI_VERSION; }

// Host-only part of oc_create: validate the layout, derive the engine constants and build the table
// image.  Needs no GPU (also used by the compile-only JIT check).
static int prepare_engine(const oc_layout_params *p, int64_t n_kitchens, oc_engine *e, std::vector<uint32_t> &tabs) {
    if (n_kitchens < 1) return fail(OC_ERR_INVALID_ARG, "oc_create: n_kitchens must be >= 1 (got %lld)", (long long)n_kitchens);
    if (p->num_players < 1 || p->num_players > OC_MAX_PLAYERS)
        return fail(OC_ERR_UNSUPPORTED, "oc_create: 1..%d players are supported (got %d)", OC_MAX_PLAYERS, p->num_players);
    if (p->width < 1 || p->height < 1 || p->width * p->height > OC_MAX_TILES)
        return fail(OC_ERR_UNSUPPORTED, "oc_create: grid %dx%d outside 1..%d tiles", p->width, p->height, OC_MAX_TILES);
    const int S = p->width * p->height;
    if (p->horizon < 1) return fail(OC_ERR_INVALID_ARG, "oc_create: horizon must be >= 1");
    int n_pots = 0, n_counters = 0;
    for (int t = 0; t < S; ++t) {
        const int terr = p->terrain[t];
        if (terr < 0 || terr > 6) return fail(OC_ERR_INVALID_ARG, "oc_create: terrain[%d] = %d outside 0..6", t, terr);
        n_pots += terr == T_POT;
        n_counters += terr == T_COUNTER;
    }
    if (n_pots > kMaxPots) return fail(OC_ERR_UNSUPPORTED, "oc_create: more than %d pots", kMaxPots);
    // table image, same offsets as carve()
    tabs.assign(lds_table_dwords(S, n_pots, n_counters), 0u);
    uint32_t *t_out2 = tabs.data(), *t_terr = t_out2 + 2 * S, *t_rv = t_terr + S, *t_rt = t_rv + 16, *t_lut = t_rt + 16;
    uint32_t *t_pots = t_lut + kLutSize, *t_counters = t_pots + n_pots;
    int ip = 0, ic = 0;
    for (int t = 0; t < S; ++t) {
        const uint32_t terr = static_cast<uint32_t>(p->terrain[t]);
        const int x = t % p->width, y = t / p->width;
        // the reference relies on the border being non-AIR so that moves never leave the grid
        if ((x == 0 || y == 0 || x == p->width - 1 || y == p->height - 1) && terr == T_AIR)
            return fail(OC_ERR_INVALID_ARG, "oc_create: border tile (%d,%d) is walkable; layouts must be walled", x, y);
        t_terr[t] = terr;
        const int o = x * p->height + y;
        const uint32_t hi2 = terr == T_POT ? 0x0001u : terr == T_COUNTER ? 0x0100u : 0u;      // channels 10, 11
        t_out2[2 * o] = static_cast<uint32_t>(t) | (terr == T_POT ? 0x100u : 0u) | (hi2 << 16);
        t_out2[2 * o + 1] = terr >= T_ONION_SRC ? (1u << (8 * (terr - T_ONION_SRC))) : 0u;   // channels 12..15
        if (terr == T_POT) t_pots[ip++] = t;
        if (terr == T_COUNTER) t_counters[ic++] = t;
    }
    if (p->soup_pickup_rew < 0 || p->soup_pickup_rew > 32767 || p->placement_in_pot_rew < 0 || p->placement_in_pot_rew > 32767)
        return fail(OC_ERR_UNSUPPORTED, "oc_create: shaped rewards must be in 0..32767");
    for (uint32_t terr = 0; terr < 7; ++terr)
        for (uint32_t h = 0; h < 5; ++h)
            for (int c = 0; c < kTileClasses; ++c)
                t_lut[(terr * 5 + h) * kTileClasses + c] = interact_outcome(terr, h, c, p->soup_pickup_rew, p->placement_in_pot_rew);
    int uniform_time = p->recipe_times[0];
    for (int i = 0; i < 16; ++i) {
        if (p->recipe_times[i] < 0 || p->recipe_times[i] > 127)
            return fail(OC_ERR_UNSUPPORTED, "oc_create: recipe_times[%d] = %d outside 0..127 (tick is a signed byte)", i, p->recipe_times[i]);
        if (p->recipe_times[i] != p->recipe_times[0]) uniform_time = -1;
        t_rt[i] = static_cast<uint32_t>(p->recipe_times[i]);
        t_rv[i] = static_cast<uint32_t>(p->recipe_values[i]);
    }
    uint32_t start_posor = 0;
    for (int i = 0; i < p->num_players; ++i) {
        const int x = p->start_player_x[i], y = p->start_player_y[i];
        if (x < 0 || y < 0 || x >= p->width || y >= p->height || p->terrain[y * p->width + x] != T_AIR)
            return fail(OC_ERR_INVALID_ARG, "oc_create: start position of player %d (%d,%d) is not a free tile", i, x, y);
        if (i < 2) start_posor |= static_cast<uint32_t>(y * p->width + x) << (16 * i);
        e->start_pp[i] = static_cast<uint32_t>(y * p->width + x);
    }

    e->params = *p;
    e->n = n_kitchens;
    e->device = -1;
    e->S = S;
    e->P = p->num_players;
    e->np_path = p->num_players != 2;
    e->recq = e->np_path ? (S + 2 * e->P + 1 + 3) / 4 : (S + 4 + 3) / 4;
    e->recd = 4 * e->recq;
    e->n_pots = n_pots;
    e->n_counters = n_counters;
    e->uniform_time = uniform_time;
    for (int i = 0; i < 4; ++i) e->pots4[i] = i < n_pots ? static_cast<int>(t_pots[i]) : 0;
    e->start_posor = start_posor;
    // Default launch geometry (oc_set_tuning overrides; results never depend on it), from the round-2 interleaved A/B runs on
    // MI355X with write-through plane stores (profiles/r02_ab_geometry.log):
    //   * 16 kitchens per group, 2 passes per flush, 12 persistent wavefronts per CU wherever 16-kitchen groups fill them
    //     (>= 3072 groups): cramped_room 65 536 kitchens 11.93 vs 12.14 us with round 1's 32 / 4 / 8, asymmetric_advantages
    //     22.1 vs 23.3, coordination_ring 13.9 vs 14.6;
    //   * smaller batches: groups of at most ~360 tiles (one wavefront's critical path grows with its tiles), and never
    //     fewer than 1024 groups while groups can still shrink: cramped_room 16 384 -> 16 per group (5.94 us),
    //     8192 -> 8 (5.49), asymmetric_advantages 16 384 -> 8 (8.57 vs 9.46 with 16), 8192 -> 8 (6.6-6.8 vs 7.2-7.4 with 4);
    //   * very large batches (>= 16 384 groups, e.g. a million kitchens) stream from HBM proper and want 16 wavefronts
    //     per CU (round 1: 0.70 vs 0.64 of roofline at 2^20 kitchens).
    //   * the smallest grids (<= 24 tiles, 32 kitchens = whole 64-tile passes) with at least 1024 groups of 32: 32 per group since
    //     the full flush groups read all their staged chunks before the first store and address the stores from a scalar base
    //     (profiles/r02_ab_geometry_flush.log): cramped_room 65 536 kitchens 11.70-11.80 vs 11.90-11.95 us, 131 072 19.98 vs
    //     21.10, 32 768 7.53 vs 7.92; not at 16 384 (6.45 vs 5.84) and not on the 5x5 grids (14.2 vs 13.7).
    auto groups_at = [&](int kpw) { return (n_kitchens + kpw - 1) / kpw; };
    e->kpw = 16;
    while (e->kpw > 4 && e->kpw * e->recq > kMaxQ * kWave) e->kpw -= 4;
    if (S <= 24 && (32 * S) % kWave == 0 && 32 * e->recq <= kMaxQ * kWave && groups_at(32) >= 1024) {
        e->kpw = 32;
    } else if (n_kitchens <= 12288) {
        //   * round 6 (profiles/r06_sweep_small_batches.log: four layouts x 4096 / 8192 / 16 384 kitchens x kitchens per group x
        //     wavefronts per workgroup): the batches an 8-GPU job runs per GPU want ~2048 groups -- 2 kitchens per group at 4096
        //     kitchens, 4 at 8192 -- in workgroups of EIGHT wavefronts: asymmetric_advantages x 8192 6.55 -> 5.71 us, cramped_room x 8192
        //     4.83 -> 4.40, x 4096 4.43 -> 4.12, coordination_ring x 8192 5.32 -> 4.75, counter_circuit x 8192 5.95 -> 5.30 (at 16 384
        //     kitchens the gain is 1-4 % and not on every layout: left alone).
        int k = 16;
        while (k > 2 && groups_at(k) < 2048) k /= 2;
        while (k < 16 && (k * S * 5) % 4 != 0) k *= 2;          // (a group's first byte in a viewer plane 16-byte aligned)
        while (k > 2 && k * e->recq > kMaxQ * kWave) k /= 2;
        e->kpw = k;
        e->wg_waves = 8;
    } else if (groups_at(e->kpw) < 3072) {
        while (e->kpw > 4 && e->kpw % 8 == 0 && e->kpw * S > 360) e->kpw /= 2;
        while (e->kpw > 4 && e->kpw % 8 == 0 && groups_at(e->kpw) < 1024) e->kpw /= 2;
    }
    //   * round 4 (profiles/r04_ab_first_passes.log, 65 536 kitchens in place): a group's FIRST flush shorter than the others starts
    //     the store stream earlier, the others can then be longer -- 2 then 4 passes per flush with 32 kitchens per group:
    //     cramped_room 11.26 -> 11.03 us; 2 then 3 with 16 per group on grids of up to 32 tiles: coordination_ring 13.53 -> 13.04;
    //     larger grids stay at 2 / 2 (counter_circuit 19.58 -> 19.39 with 1 then 3, asymmetric_advantages 21.8 -> 25.1: its LDS
    //     then holds eight wavefronts per CU instead of twelve).
    const int64_t n_groups = groups_at(e->kpw);
    e->gpasses = n_groups < 1024 ? 4 : 2;
    e->first_passes = 0;
    e->encode_ilp4 = 0;
    // (four tiles per lane in flight in the four-pass flushes: 11.04 -> 10.93 us, profiles/r04_ab_ilp4.log; neutral on the other shapes)
    if (e->kpw == 32 && n_groups >= 2048) { e->gpasses = 4; e->first_passes = 2; e->encode_ilp4 = 1; }     // (32 768 kitchens: 7.10 -> 7.69 us, left alone)
    else if (n_groups >= 3072 && e->kpw == 16 && S <= 32) { e->gpasses = 3; e->first_passes = 2; }
    e->waves_per_cu = n_groups >= 16384 ? 16 : n_groups < 1024 ? 8 : 12;
    e->kpp = kpp_for(S, e->gpasses);
    e->num_cus = 256;
    // the persistent wavefronts of a CU must all fit its 160 KB of LDS, or the surplus ones queue behind the resident ones
    while (e->waves_per_cu > 4 && lds_bytes(e, e->kpw, e->gpasses) * e->waves_per_cu > 160 * 1024) e->waves_per_cu -= 4;
    { const char *ab = OC_DIAG_ENV("OC_ABLATE"); e->ablate = ab ? atoi(ab) : 0; }
    e->cu_budget = 0;
    e->tuned_by_user = false;
    e->d_state = nullptr;
    e->d_tabs = nullptr;
    e->d_trace = nullptr;
    e->d_fold_ws = nullptr;
    e->d_fold_args = nullptr;
    e->ev0 = e->ev1 = nullptr;
    e->arch[0] = 0;
    e->last_obs = nullptr;
    snprintf(e->jit_status, sizeof(e->jit_status), "not built");
    return OC_OK;
}

static int create_impl(const oc_layout_params *p, int64_t n_kitchens, int device_id, oc_engine **out);

int oc_create(const oc_layout_params *p, int64_t n_kitchens, int device_id, oc_engine **out) {
    // nothing may propagate across the C boundary (an allocation failure on absurd arguments included)
    try {
        return create_impl(p, n_kitchens, device_id, out);
    } catch (const std::exception &ex) {
        return fail(OC_ERR_INVALID_ARG, "oc_create: %s", ex.what());
    } catch (...) {
        return fail(OC_ERR_INVALID_ARG, "oc_create: unexpected failure");
    }
}

static int create_impl(const oc_layout_params *p, int64_t n_kitchens, int device_id, oc_engine **out) {
    if (!p || !out) return fail(OC_ERR_INVALID_ARG, "oc_create: NULL argument");
    *out = nullptr;
    oc_engine *e = new (std::nothrow) oc_engine();
    if (!e) return fail(OC_ERR_INVALID_ARG, "oc_create: out of host memory");
    std::vector<uint32_t> tabs;
    if (int rc = prepare_engine(p, n_kitchens, e, tabs)) { delete e; return rc; }

    int ndev = 0;
    if (hipGetDeviceCount(&ndev) != hipSuccess || ndev == 0) {
        delete e;
        return fail(OC_ERR_NO_DEVICE, "oc_create: no HIP device visible (this engine has no CPU fallback)");
    }
    if (device_id < 0 || device_id >= ndev) { delete e; return fail(OC_ERR_INVALID_ARG, "oc_create: device_id %d outside 0..%d", device_id, ndev - 1); }
    e->device = device_id;
    const OcDeviceScope on_device(device_id);          // the caller's current device is put back on return
    hipDeviceProp_t prop;
    hipError_t err = on_device.ok ? hipSuccess : hipErrorInvalidDevice;
    if (err == hipSuccess) err = hipGetDeviceProperties(&prop, device_id);
    if (err == hipSuccess) {
        e->num_cus = prop.multiProcessorCount > 0 ? prop.multiProcessorCount : 256;
        snprintf(e->arch, sizeof(e->arch), "%s", prop.gcnArchName);
    }
    if (err == hipSuccess) err = hipMalloc(reinterpret_cast<void **>(&e->d_state), static_cast<size_t>(n_kitchens) * e->recq * sizeof(uint4));
    if (err == hipSuccess) err = hipMalloc(reinterpret_cast<void **>(&e->d_tabs), tabs.size() * sizeof(uint32_t));
    if (err == hipSuccess) err = hipMemcpy(e->d_tabs, tabs.data(), tabs.size() * sizeof(uint32_t), hipMemcpyHostToDevice);
    if (err == hipSuccess) err = hipEventCreate(&e->ev0);
    if (err == hipSuccess) err = hipEventCreate(&e->ev1);
    if (err != hipSuccess) {
        fail(OC_ERR_HIP, "oc_create: device set-up failed: %s", hipGetErrorString(err));
        oc_destroy(e);
        return OC_ERR_HIP;
    }
    if (e->np_path) snprintf(e->jit_status, sizeof(e->jit_status), "%d-player group kernel, one launch per step (ahead of time)", e->P);
    else jit_build(e);
    int rc = oc_reset_all(e, nullptr, nullptr);
    if (rc == OC_OK && hipDeviceSynchronize() != hipSuccess) rc = fail(OC_ERR_HIP, "oc_create: start-state fill failed");
    if (rc != OC_OK) { oc_destroy(e); return rc; }
    *out = e;
    return OC_OK;
}

int oc_destroy(oc_engine *e) {
    if (!e) return OC_OK;
    const OcDeviceScope on_device(e->device);
    if (e->d_state) (void)hipFree(e->d_state);
    if (e->d_state_alt) (void)hipFree(e->d_state_alt);
    if (e->d_tabs) (void)hipFree(e->d_tabs);
    if (e->d_trace) (void)hipFree(e->d_trace);
    if (e->d_fold_ws) (void)hipFree(e->d_fold_ws);
    if (e->d_fold_args) (void)hipFree(e->d_fold_args);
    jit_unload(e);
    if (e->ev0) (void)hipEventDestroy(e->ev0);
    if (e->ev1) (void)hipEventDestroy(e->ev1);
    delete e;
    return OC_OK;
}

int oc_step(oc_engine *e, const void *d_actions, int action_dtype, int8_t *d_obs, int32_t *d_reward, int32_t *d_done,
            void *d_records, void *stream) {
    if (int rc = check_engine(e)) return rc;
    OC_ON_ENGINE_DEVICE(e);
    note_stream(e, static_cast<hipStream_t>(stream));
    if (!d_actions || !d_obs || !d_reward || !d_done) return fail(OC_ERR_INVALID_ARG, "oc_step: NULL device buffer");
    if (action_dtype != OC_ACT_I32 && action_dtype != OC_ACT_I64) return fail(OC_ERR_INVALID_ARG, "oc_step: bad action dtype %d", action_dtype);
    if (reinterpret_cast<uintptr_t>(d_obs) % 4) return fail(OC_ERR_INVALID_ARG, "oc_step: obs buffer must be 4-byte aligned");
    if (reinterpret_cast<uintptr_t>(d_records) % 16) return fail(OC_ERR_INVALID_ARG, "oc_step: the record destination must be 16-byte aligned");
    return step_impl(e, d_actions, action_dtype, d_obs, d_reward, d_done, d_records, static_cast<hipStream_t>(stream));
}

/* The step with the two players' actions in two buffers (round 6).  The drop-in classes get the ego's action tensor from the caller
 * and the partner's from its agent (VectorMultiAgentEnv.step, pantheonrl_extension/vectorenv.py:171-193) and used to assemble the
 * [P, N, 1] tensor the simulator wants with a torch.stack -- 7 of the 18 us of a Python-driven step (tools/exp_drop_in_breakdown.py).
 * Here the kernel reads the two buffers where they are.  In-place destinations of 2-player engines on the specialised kernel only;
 * anything else returns OC_ERR_UNSUPPORTED and the caller assembles and calls oc_step. */
int oc_step_players(oc_engine *e, const void *const *d_actions, int action_dtype, int8_t *d_obs, int32_t *d_reward, int32_t *d_done, void *stream) {
    if (int rc = check_engine(e)) return rc;
    if (!d_actions || !d_actions[0] || !d_actions[1] || !d_obs || !d_reward || !d_done) return fail(OC_ERR_INVALID_ARG, "oc_step_players: NULL device buffer");
    if (action_dtype != OC_ACT_I32 && action_dtype != OC_ACT_I64) return fail(OC_ERR_INVALID_ARG, "oc_step_players: bad action dtype %d", action_dtype);
    if (reinterpret_cast<uintptr_t>(d_obs) % 4) return fail(OC_ERR_INVALID_ARG, "oc_step_players: obs buffer must be 4-byte aligned");
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (e->np_path || !wide_stores() || !e->jit.mod || e->jit.kpw != e->kpw || e->jit.gpasses != e->gpasses || e->jit.xw.sum ||
        (e->last_obs != nullptr && d_obs != e->last_obs) || 2 * e->n * e->S * kChannels > kStreamInPlaceBytes)
        return fail(OC_ERR_UNSUPPORTED, "oc_step_players: in-place steps of 2-player engines on the specialised kernel only");
    OC_ON_ENGINE_DEVICE(e);
    note_stream(e, s);
    if (!ensure_2p_module(e, own_tuning(e))) return fail(OC_ERR_UNSUPPORTED, "oc_step_players: the two-buffer entry points could not be built");
    StepArgs a = make_args(e, e->d_state, e->n, d_actions[0], d_obs, d_reward, d_done);
    a.actions1 = d_actions[1];
    if (a.n_kitchens == 0) return OC_OK;
    const unsigned grid = static_cast<unsigned>(min(static_cast<int64_t>(a.n_groups), static_cast<int64_t>(e->waves_per_cu) * launch_cus(e)));
    OC_HIP(launch_jit(e->jit_2p.fn[action_dtype == OC_ACT_I64 ? JIT_STEP_I64_V16_2P : JIT_STEP_I32_V16_2P], a, grid, lds_bytes(e, a.kpw, a.gpasses), s, e->jit_2p.wg, true));
    e->last_obs = d_obs;
    return OC_OK;
}

int oc_observe(oc_engine *e, int8_t *d_obs, void *stream) {
    if (int rc = check_engine(e)) return rc;
    OC_ON_ENGINE_DEVICE(e);
    note_stream(e, static_cast<hipStream_t>(stream));
    if (!d_obs) return fail(OC_ERR_INVALID_ARG, "oc_observe: NULL obs buffer");
    if (reinterpret_cast<uintptr_t>(d_obs) % 4) return fail(OC_ERR_INVALID_ARG, "oc_observe: obs buffer must be 4-byte aligned");
    if (e->np_path)
        return np_encode(e, reinterpret_cast<const uint32_t *>(e->d_state), e->n, d_obs, e->n * e->S * (5 * e->P + 10), static_cast<hipStream_t>(stream));
    const StepArgs a = make_args(e, e->d_state, e->n, nullptr, d_obs, nullptr, nullptr);
    return launch<false, false>(e, a, static_cast<hipStream_t>(stream));
}

int oc_encode_states_strided(oc_engine *e, const void *d_states, int64_t n, int8_t *d_obs, int64_t obs_player_stride,
                             void *stream) {
    if (int rc = check_engine(e)) return rc;
    if (!d_states || !d_obs || n < 0) return fail(OC_ERR_INVALID_ARG, "oc_encode_states: bad argument");
    OC_ON_ENGINE_DEVICE(e);
    if (reinterpret_cast<uintptr_t>(d_states) % 16) return fail(OC_ERR_INVALID_ARG, "oc_encode_states: state block must be 16-byte aligned");
    // (the N-player encoder checks every block's destination and falls back to byte stores, exactly as for oc_step / oc_observe,
    // whose viewer stride n * S * (5P + 10) is odd for odd n, S and P: no alignment to ask for there)
    if (!e->np_path && (reinterpret_cast<uintptr_t>(d_obs) % 4 || obs_player_stride % 4))
        return fail(OC_ERR_INVALID_ARG, "oc_encode_states: obs buffer/stride must be 4-byte aligned");
    if (obs_player_stride < n * e->S * (5 * e->P + 10)) return fail(OC_ERR_INVALID_ARG, "oc_encode_states: viewer planes would overlap");
    if (e->np_path) return np_encode(e, static_cast<const uint32_t *>(d_states), n, d_obs, obs_player_stride, static_cast<hipStream_t>(stream));
    StepArgs a = make_args(e, const_cast<uint4 *>(static_cast<const uint4 *>(d_states)), n, nullptr, d_obs, nullptr, nullptr);
    a.obs_player_stride = obs_player_stride;
    return launch<false, false>(e, a, static_cast<hipStream_t>(stream));
}

int oc_encode_states(oc_engine *e, const void *d_states, int64_t n, int8_t *d_obs, void *stream) {
    if (int rc = check_engine(e)) return rc;
    return oc_encode_states_strided(e, d_states, n, d_obs, n * e->S * (5 * e->P + 10), stream);
}

int oc_encode_trajectory(oc_engine *e, const void *d_states, int64_t n, int64_t T, int64_t state_step_stride, int8_t *d_obs,
                         int64_t obs_player_stride, int64_t obs_step_stride, void *stream) {
    if (int rc = check_engine(e)) return rc;
    if (!d_states || !d_obs || n < 0 || T < 0) return fail(OC_ERR_INVALID_ARG, "oc_encode_trajectory: bad argument");
    if (e->np_path) {
        // kitchens with 1, 3 or 4 players: the group kernel over all T blocks of records in ONE launch (round 5; a launch per time step before)
        if (reinterpret_cast<uintptr_t>(d_states) % 4 || state_step_stride % 4 || state_step_stride < n * e->recd * 4)
            return fail(OC_ERR_INVALID_ARG, "oc_encode_trajectory: record blocks must be 4-byte aligned and must not overlap");
        if (obs_player_stride < n * e->S * (5 * e->P + 10)) return fail(OC_ERR_INVALID_ARG, "oc_encode_trajectory: viewer planes would overlap");
        if (T == 0 || n == 0) return OC_OK;
        OC_ON_ENGINE_DEVICE(e);
        oc_np::NpArgs a = np_args(e, const_cast<uint32_t *>(static_cast<const uint32_t *>(d_states)), n, nullptr, 0, d_obs, obs_player_stride, nullptr, nullptr);
        a.items = T; a.state_item_stride = state_step_stride / 4; a.obs_item_stride = obs_step_stride;
        return np_launch<false>(e, a, static_cast<hipStream_t>(stream));
    }
    if (reinterpret_cast<uintptr_t>(d_states) % 16 || state_step_stride % 16 || state_step_stride < n * e->recq * 16)
        return fail(OC_ERR_INVALID_ARG, "oc_encode_trajectory: record blocks must be 16-byte aligned and must not overlap");
    if (reinterpret_cast<uintptr_t>(d_obs) % 4 || obs_player_stride % 4 || obs_step_stride % 4)
        return fail(OC_ERR_INVALID_ARG, "oc_encode_trajectory: obs buffer/strides must be 4-byte aligned");
    if (obs_player_stride < n * e->S * kChannels) return fail(OC_ERR_INVALID_ARG, "oc_encode_trajectory: viewer planes would overlap");
    OC_ON_ENGINE_DEVICE(e);
    StepArgs a = make_args(e, const_cast<uint4 *>(static_cast<const uint4 *>(d_states)), n, nullptr, d_obs, nullptr, nullptr);
    a.obs_player_stride = obs_player_stride;
    a.state_batch_stride = state_step_stride / 16;
    a.obs_batch_stride = obs_step_stride;
    return launch_observe_batch(e, a, T, static_cast<hipStream_t>(stream));
}

int oc_group_create(oc_engine *const *engines, int32_t n_engines, oc_group **out) {
    if (!engines || !out || n_engines < 1 || n_engines > kMaxSegments)
        return fail(OC_ERR_INVALID_ARG, "oc_group_create: 1..%d engines", kMaxSegments);
    *out = nullptr;
    for (int i = 0; i < n_engines; ++i) {
        if (!engines[i]) return fail(OC_ERR_INVALID_ARG, "oc_group_create: engine %d is NULL", i);
        if (engines[i]->device != engines[0]->device) return fail(OC_ERR_INVALID_ARG, "oc_group_create: the engines of a group must live on one GPU");
        for (int j = 0; j < i; ++j)
            if (engines[j] == engines[i]) return fail(OC_ERR_INVALID_ARG, "oc_group_create: engine %d is listed twice", i);
    }
    oc_group *g = new (std::nothrow) oc_group();
    if (!g) return fail(OC_ERR_INVALID_ARG, "oc_group_create: out of host memory");
    g->engines.assign(engines, engines + n_engines);
    g->device = engines[0]->device;
    g->waves_per_cu = 12;
    g->num_cus = engines[0]->num_cus;
    g->mod = nullptr;
    g->shmem = 0;
    g->last_obs0 = nullptr;
    snprintf(g->status, sizeof(g->status), "not built");
    const OcDeviceScope on_device(g->device);
    bool any_np = false;
    for (int i = 0; i < n_engines; ++i) any_np = any_np || engines[i]->np_path;
    if (any_np) {
        // kitchens with 1, 3 or 4 players have no specialised body to put into a group module: the group then steps its engines one
        // launch (pair) after the other -- same results, same calls
        g->tunings.assign(n_engines, Tuning{0, 0, 0});
        g->blocks.assign(n_engines, 0);
        g->layout_of_seg.assign(n_engines, 0);
        snprintf(g->status, sizeof(g->status), "one launch per engine (%d engines; kitchens with other than 2 players run on the plain kernels)", n_engines);
        *out = g;
        return OC_OK;
    }
    if (int rc = group_plan(g, nullptr, 0, 0)) { delete g; return rc; }
    group_build(g);
    *out = g;
    return OC_OK;
}

int oc_group_destroy(oc_group *g) {
    if (!g) return OC_OK;
    const OcDeviceScope on_device(g->device);
    (void)hipDeviceSynchronize();                 // the module may still be executing
    group_unload(g);
    delete g;
    return OC_OK;
}

int32_t oc_group_size(const oc_group *g) { return g ? static_cast<int32_t>(g->engines.size()) : 0; }
const char *oc_group_build_info(const oc_group *g) { return g ? g->status : ""; }

int oc_group_set_tuning(oc_group *g, const int32_t *kitchens_per_wave, int passes_per_flush, int waves_per_cu) {
    if (int rc = check_group(g)) return rc;
    if (waves_per_cu < 0 || waves_per_cu > 32) return fail(OC_ERR_INVALID_ARG, "oc_group_set_tuning: waves_per_cu must be in 1..32 (0 keeps it)");
    for (const oc_engine *e : g->engines)
        if (e->np_path) return OC_OK;                     // one launch per engine: no joint geometry to tune
    OC_ON_GROUP_DEVICE(g);
    const std::vector<Tuning> old_t = g->tunings;
    const std::vector<int> old_b = g->blocks;
    const int old_w = g->waves_per_cu;
    const size_t old_s = g->shmem;
    if (int rc = group_plan(g, kitchens_per_wave, passes_per_flush, waves_per_cu)) {
        g->tunings = old_t; g->blocks = old_b; g->waves_per_cu = old_w; g->shmem = old_s;
        return rc;
    }
    OC_HIP(hipDeviceSynchronize());               // the old module may still be executing
    group_build(g);
    return OC_OK;
}

int oc_group_step(oc_group *g, const void *const *d_actions, int action_dtype, int8_t *const *d_obs, int32_t *const *d_reward,
                  int32_t *const *d_done, void *const *d_records, void *stream) {
    if (int rc = check_group(g)) return rc;
    if (!d_actions || !d_obs || !d_reward || !d_done) return fail(OC_ERR_INVALID_ARG, "oc_group_step: NULL pointer table");
    if (action_dtype != OC_ACT_I32 && action_dtype != OC_ACT_I64) return fail(OC_ERR_INVALID_ARG, "oc_group_step: bad action dtype %d", action_dtype);
    const int n = static_cast<int>(g->engines.size());
    const bool vec16 = wide_stores();
    for (int i = 0; i < n; ++i) {
        if (!d_actions[i] || !d_obs[i] || !d_reward[i] || !d_done[i]) return fail(OC_ERR_INVALID_ARG, "oc_group_step: NULL device buffer for engine %d", i);
        // (kitchens with other than 2 players run on the plain kernels, whose encoder takes any alignment -- as oc_step does)
        if (!g->engines[i]->np_path && reinterpret_cast<uintptr_t>(d_obs[i]) % 4) return fail(OC_ERR_INVALID_ARG, "oc_group_step: obs buffers must be 4-byte aligned");
        if (d_records && reinterpret_cast<uintptr_t>(d_records[i]) % 16) return fail(OC_ERR_INVALID_ARG, "oc_group_step: record destinations must be 16-byte aligned");
    }
    OC_ON_GROUP_DEVICE(g);
    for (oc_engine *ge : g->engines) note_stream(ge, static_cast<hipStream_t>(stream));
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (!g->mod || !vec16) {                      // no group module (OC_NO_JIT, hiprtc failure; dword-store diagnostics): one launch per engine
        for (int i = 0; i < n; ++i)
            if (int rc = step_impl(g->engines[i], d_actions[i], action_dtype, d_obs[i], d_reward[i], d_done[i], d_records ? d_records[i] : nullptr, s)) return rc;
        return OC_OK;
    }
    GroupArgs m;
    for (int i = 0; i < n; ++i) {
        oc_engine *e = g->engines[i];
        m.seg[i] = make_args(e, g->tunings[i], e->d_state, e->n, d_actions[i], d_obs[i], d_reward[i], d_done[i]);
        m.seg[i].rec_out = d_records ? static_cast<uint4 *>(d_records[i]) : nullptr;
        m.seg[i].trace = nullptr;
        e->last_obs = d_obs[i];
    }
    for (int i = n; i < kMaxSegments; ++i) m.seg[i] = m.seg[0];
    // a destination that differs from the previous step's is a trajectory slot: stream it past the caches (see store16)
    const bool nt = d_obs[0] != g->last_obs0;
    g->last_obs0 = d_obs[0];
    const bool pl = nt && g->engines[0]->planes_read_next;           // (a group rollout with the policies in the loop sets it on every engine)
    const int idx = action_dtype == OC_ACT_I64 ? (pl ? GJIT_STEP_I64_PL : nt ? GJIT_STEP_I64_NT : GJIT_STEP_I64)
                                               : (pl ? GJIT_STEP_I32_PL : nt ? GJIT_STEP_I32_NT : GJIT_STEP_I32);
    return group_launch(g, idx, m, s);
}

int oc_group_observe(oc_group *g, int8_t *const *d_obs, void *stream) {
    if (int rc = check_group(g)) return rc;
    if (!d_obs) return fail(OC_ERR_INVALID_ARG, "oc_group_observe: NULL pointer table");
    const int n = static_cast<int>(g->engines.size());
    const bool vec16 = wide_stores();
    for (int i = 0; i < n; ++i)
        if (!d_obs[i] || (!g->engines[i]->np_path && reinterpret_cast<uintptr_t>(d_obs[i]) % 4))
            return fail(OC_ERR_INVALID_ARG, "oc_group_observe: NULL or misaligned obs buffer for engine %d", i);
    OC_ON_GROUP_DEVICE(g);
    for (oc_engine *ge : g->engines) note_stream(ge, static_cast<hipStream_t>(stream));
    if (!g->mod || !vec16) {
        for (int i = 0; i < n; ++i)
            if (int rc = oc_observe(g->engines[i], d_obs[i], stream)) return rc;
        return OC_OK;
    }
    GroupArgs m;
    for (int i = 0; i < n; ++i) {
        oc_engine *e = g->engines[i];
        m.seg[i] = make_args(e, g->tunings[i], e->d_state, e->n, nullptr, d_obs[i], nullptr, nullptr);
        m.seg[i].trace = nullptr;
    }
    for (int i = n; i < kMaxSegments; ++i) m.seg[i] = m.seg[0];
    return group_launch(g, GJIT_OBS, m, static_cast<hipStream_t>(stream));
}

int oc_group_rollout_timed(oc_group *g, const void *const *d_actions, int action_dtype, int64_t T_act, int64_t T, int8_t *const *d_obs,
                           int32_t *const *d_reward, int32_t *const *d_done, void *stream, float *elapsed_ms) {
    if (int rc = check_group(g)) return rc;
    if (!elapsed_ms || !d_actions || T_act < 1 || T < 0) return fail(OC_ERR_INVALID_ARG, "oc_group_rollout_timed: bad argument");
    if (action_dtype != OC_ACT_I32 && action_dtype != OC_ACT_I64) return fail(OC_ERR_INVALID_ARG, "oc_group_rollout_timed: bad action dtype %d", action_dtype);
    OC_ON_GROUP_DEVICE(g);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int n = static_cast<int>(g->engines.size());
    const size_t asz = action_dtype == OC_ACT_I64 ? 8 : 4;
    std::vector<const void *> act(n);
    oc_engine *e0 = g->engines[0];
    OC_HIP(hipEventRecord(e0->ev0, s));
    for (int64_t t = 0; t < T; ++t) {
        for (int i = 0; i < n; ++i)
            act[i] = static_cast<const char *>(d_actions[i]) + static_cast<size_t>(t % T_act) * g->engines[i]->P * g->engines[i]->n * asz;
        if (int rc = oc_group_step(g, act.data(), action_dtype, d_obs, d_reward, d_done, nullptr, stream)) return rc;
    }
    OC_HIP(hipEventRecord(e0->ev1, s));
    OC_HIP(wait_event(e0->ev1));
    OC_HIP(hipEventElapsedTime(elapsed_ms, e0->ev0, e0->ev1));
    return OC_OK;
}

int oc_reset_all(oc_engine *e, int8_t *d_obs, void *stream) {
    if (int rc = check_engine(e)) return rc;
    OC_ON_ENGINE_DEVICE(e);
    note_stream(e, static_cast<hipStream_t>(stream));
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (e->np_path) {
        const int64_t words = e->n * e->recd;
        hipLaunchKernelGGL(oc_np::np_fill_start_kernel, dim3(static_cast<unsigned>((words + 255) / 256)), dim3(256), 0, s, reinterpret_cast<uint32_t *>(e->d_state),
                           e->n, e->S, e->P, e->recd, e->start_pp[0], e->start_pp[1], e->start_pp[2], e->start_pp[3]);
        OC_HIP(hipGetLastError());
        if (d_obs) return oc_observe(e, d_obs, stream);
        return OC_OK;
    }
    const int64_t chunks = e->n * e->recq;
    const unsigned grid = static_cast<unsigned>((chunks + 255) / 256);
    hipLaunchKernelGGL(oc_fill_start_kernel, dim3(grid), dim3(256), 0, s, e->d_state, (int64_t)0, e->n, e->recq, e->S, e->start_posor);
    OC_HIP(hipGetLastError());
    if (d_obs) return oc_observe(e, d_obs, stream);
    return OC_OK;
}

int oc_episode_control(oc_engine *e, const int32_t *d_reset_mask, const int32_t *d_timesteps, void *stream) {
    if (int rc = check_engine(e)) return rc;
    OC_ON_ENGINE_DEVICE(e);
    note_stream(e, static_cast<hipStream_t>(stream));
    if (!d_reset_mask && !d_timesteps) return OC_OK;
    if (e->np_path) {
        hipLaunchKernelGGL(oc_np::np_episode_control_kernel, dim3(static_cast<unsigned>((e->n + 255) / 256)), dim3(256), 0, static_cast<hipStream_t>(stream),
                           reinterpret_cast<uint32_t *>(e->d_state), e->n, e->S, e->P, e->recd, e->params.horizon, e->start_pp[0], e->start_pp[1],
                           e->start_pp[2], e->start_pp[3], d_reset_mask, d_timesteps);
        OC_HIP(hipGetLastError());
        return OC_OK;
    }
    const int64_t chunks = e->n * e->recq;
    hipLaunchKernelGGL(oc_episode_control_kernel, dim3(static_cast<unsigned>((chunks + 255) / 256)), dim3(256), 0,
                       static_cast<hipStream_t>(stream), e->d_state, e->n, e->recq, e->S, e->start_posor, e->params.horizon,
                       d_reset_mask, d_timesteps);
    OC_HIP(hipGetLastError());
    return OC_OK;
}

int oc_rollout(oc_engine *e, const void *d_actions, int action_dtype, int64_t T_act, int64_t T, int8_t *d_obs,
               int64_t obs_step_stride, int32_t *d_reward, int64_t reward_step_stride, int32_t *d_done,
               int64_t done_step_stride, void *d_records, int64_t records_step_stride, void *stream) {
    if (int rc = check_engine(e)) return rc;
    OC_ON_ENGINE_DEVICE(e);
    note_stream(e, static_cast<hipStream_t>(stream));
    if (!d_actions || !d_obs || !d_reward || !d_done || T_act < 1 || T < 0)
        return fail(OC_ERR_INVALID_ARG, "oc_rollout: bad argument");
    if (action_dtype != OC_ACT_I32 && action_dtype != OC_ACT_I64) return fail(OC_ERR_INVALID_ARG, "oc_rollout: bad action dtype %d", action_dtype);
    if (!e->np_path && (reinterpret_cast<uintptr_t>(d_obs) % 4 || obs_step_stride % 4))
        return fail(OC_ERR_INVALID_ARG, "oc_rollout: obs buffer/stride must be 4-byte aligned");
    if (d_records && (reinterpret_cast<uintptr_t>(d_records) % 16 || records_step_stride % 16 || records_step_stride < 0))
        return fail(OC_ERR_INVALID_ARG, "oc_rollout: record destination / stride must be 16-byte aligned");
    const size_t asz = action_dtype == OC_ACT_I64 ? 8 : 4;
    hipStream_t s = static_cast<hipStream_t>(stream);
    for (int64_t t = 0; t < T; ++t) {
        const char *act = static_cast<const char *>(d_actions) + static_cast<size_t>(t % T_act) * e->P * e->n * asz;   // slice t % T_act of [T_act][P][N]
        if (int rc = step_impl(e, act, action_dtype, d_obs + t * obs_step_stride, d_reward + t * reward_step_stride,
                               d_done + t * done_step_stride, d_records ? static_cast<char *>(d_records) + t * records_step_stride : nullptr, s))
            return rc;
    }
    return OC_OK;
}

int oc_rollout_timed(oc_engine *e, const void *d_actions, int action_dtype, int64_t T_act, int64_t T, int8_t *d_obs,
                     int32_t *d_reward, int32_t *d_done, void *stream, float *elapsed_ms) {
    if (int rc = check_engine(e)) return rc;
    OC_ON_ENGINE_DEVICE(e);
    if (!elapsed_ms) return fail(OC_ERR_INVALID_ARG, "oc_rollout_timed: NULL elapsed_ms");
    hipStream_t s = static_cast<hipStream_t>(stream);
    OC_HIP(hipEventRecord(e->ev0, s));
    if (int rc = oc_rollout(e, d_actions, action_dtype, T_act, T, d_obs, 0, d_reward, 0, d_done, 0, nullptr, 0, stream)) return rc;
    OC_HIP(hipEventRecord(e->ev1, s));
    OC_HIP(wait_event(e->ev1));
    OC_HIP(hipEventElapsedTime(elapsed_ms, e->ev0, e->ev1));
    return OC_OK;
}

int oc_rollout_fused(oc_engine *e, const void *d_actions, int action_dtype, int64_t T_act, int64_t T, uint32_t rng_seed,
                     uint32_t rng_t0, int8_t *d_obs, int64_t obs_step_stride, int32_t *d_reward, int64_t reward_step_stride,
                     int32_t *d_done, int64_t done_step_stride, void *d_records, int64_t records_step_stride, void *stream) {
    if (int rc = check_engine(e)) return rc;
    OC_ON_ENGINE_DEVICE(e);
    note_stream(e, static_cast<hipStream_t>(stream));
    if (!d_obs || !d_reward || !d_done || T < 0 || T > 0x7fffffff) return fail(OC_ERR_INVALID_ARG, "oc_rollout_fused: bad argument");
    if (d_actions && (T_act < 1 || T_act > 0x7fffffff || (action_dtype != OC_ACT_I32 && action_dtype != OC_ACT_I64)))
        return fail(OC_ERR_INVALID_ARG, "oc_rollout_fused: bad action tape (1 .. 2^31 - 1 slices, i32 or i64)");
    if (d_records && (reinterpret_cast<uintptr_t>(d_records) % 16 || records_step_stride % 16 || records_step_stride < 0))
        return fail(OC_ERR_INVALID_ARG, "oc_rollout_fused: record destination / stride must be 16-byte aligned");
    if (e->np_path) {
        // kitchens with 1, 3 or 4 players: the same rollout as T step launches (a tape only: the built-in action stream is defined
        // for two players).  Results are those of T calls of oc_step either way.
        if (!d_actions) return fail(OC_ERR_UNSUPPORTED, "oc_rollout_fused: the built-in action stream is 2-player; pass a tape for %d-player kitchens", e->P);
        if (T == 0) return OC_OK;
        // ONE launch for the T steps here too (round 5): every group's records stay in LDS between the steps
        oc_np::NpArgs a = np_args(e, reinterpret_cast<uint32_t *>(e->d_state), e->n, d_actions, action_dtype == OC_ACT_I64 ? 1 : 0, d_obs,
                                  e->n * e->S * (5 * e->P + 10), d_reward, d_done);
        a.rec_out = static_cast<uint32_t *>(d_records);
        a.n_steps = static_cast<int32_t>(T); a.tape_steps = static_cast<int32_t>(T_act);
        a.obs_step_stride = obs_step_stride; a.reward_step_stride = reward_step_stride; a.done_step_stride = done_step_stride;
        a.rec_step_stride = records_step_stride / 4;
        return np_launch<true>(e, a, static_cast<hipStream_t>(stream));
    }
    if (reinterpret_cast<uintptr_t>(d_obs) % 4 || obs_step_stride % 4 || obs_step_stride < 0)
        return fail(OC_ERR_INVALID_ARG, "oc_rollout_fused: obs buffer/stride must be 4-byte aligned");
    StepArgs a = make_args(e, fused_tuning(e), e->d_state, e->n, d_actions, d_obs, d_reward, d_done);
    a.n_steps = static_cast<int32_t>(T);
    a.tape_steps = static_cast<int32_t>(d_actions ? T_act : 1);
    a.action_step_stride = 2 * e->n;
    a.obs_step_stride = obs_step_stride;
    a.reward_step_stride = reward_step_stride;
    a.done_step_stride = done_step_stride;
    a.rng_seed = rng_seed;
    a.rng_t0 = rng_t0;
    a.rec_out = static_cast<uint4 *>(d_records);
    a.rec_step_stride = records_step_stride / 16;
    return launch_fused(e, a, d_actions && action_dtype == OC_ACT_I64, static_cast<hipStream_t>(stream));
}

uint32_t oc_synthetic_action(uint32_t seed, uint32_t kitchen, uint32_t step, uint32_t player) {
    return oc_hash_action(seed, kitchen, step, player);
}

int64_t oc_state_record_bytes(const oc_engine *e) { return e ? static_cast<int64_t>(e->recq) * 16 : 0; }
int64_t oc_num_kitchens(const oc_engine *e) { return e ? e->n : 0; }
int oc_device_id(const oc_engine *e) { return e ? e->device : -1; }

int oc_obs_shape(const oc_engine *e, int64_t shape5[5]) {
    if (int rc = check_engine(e)) return rc;
    if (!shape5) return fail(OC_ERR_INVALID_ARG, "oc_obs_shape: NULL output");
    shape5[0] = e->P; shape5[1] = e->n; shape5[2] = e->params.width; shape5[3] = e->params.height; shape5[4] = 5 * e->P + 10;
    return OC_OK;
}

static int check_range(const oc_engine *e, int64_t first, int64_t count, const char *who) {
    if (first < 0 || count < 0 || first + count > e->n)
        return fail(OC_ERR_INVALID_ARG, "%s: range [%lld, %lld) outside 0..%lld", who, (long long)first, (long long)(first + count), (long long)e->n);
    return OC_OK;
}

int oc_get_state(oc_engine *e, int64_t first, int64_t count, void *host_dst) {
    if (int rc = check_engine(e)) return rc;
    if (!host_dst) return fail(OC_ERR_INVALID_ARG, "oc_get_state: NULL destination");
    if (int rc = check_range(e, first, count, "oc_get_state")) return rc;
    OC_ON_ENGINE_DEVICE(e);
    OC_HIP(hipDeviceSynchronize());
    OC_HIP(hipMemcpy(host_dst, e->d_state + first * e->recq, static_cast<size_t>(count) * e->recq * 16, hipMemcpyDeviceToHost));
    return OC_OK;
}

int oc_set_state(oc_engine *e, int64_t first, int64_t count, const void *host_src) {
    if (int rc = check_engine(e)) return rc;
    if (!host_src) return fail(OC_ERR_INVALID_ARG, "oc_set_state: NULL source");
    if (int rc = check_range(e, first, count, "oc_set_state")) return rc;
    // reject records the kernels could fault on: positions must index real tiles
    const uint32_t *w = static_cast<const uint32_t *>(host_src);
    for (int64_t k = 0; k < count; ++k) {
        const int W = e->params.width, H = e->params.height;
        auto interior = [&](int p) { const int x = p % W, y = p / W; return p < e->S && x > 0 && y > 0 && x < W - 1 && y < H - 1; };
        bool ok = true;
        if (e->np_path) {
            for (int i = 0; i < e->P; ++i) {
                const uint32_t pp = w[k * e->recd + e->S + i];
                ok = ok && interior(pp & 0xff) && ((pp >> 8) & 0xff) <= 3;
            }
        } else {
            const uint32_t posor = w[k * e->recq * 4 + e->S];
            ok = interior(posor & 0xff) && interior((posor >> 16) & 0xff) && ((posor >> 8) & 0xff) <= 3 && (posor >> 24) <= 3;
        }
        if (!ok) return fail(OC_ERR_INVALID_ARG, "oc_set_state: record %lld has a player off the interior grid or a bad orientation", (long long)(first + k));
    }
    OC_ON_ENGINE_DEVICE(e);
    OC_HIP(hipDeviceSynchronize());
    OC_HIP(hipMemcpy(e->d_state + first * e->recq, host_src, static_cast<size_t>(count) * e->recq * 16, hipMemcpyHostToDevice));
    return OC_OK;
}

int oc_export_states(oc_engine *e, int64_t first, int64_t count, void *d_dst, void *stream) {
    if (int rc = check_engine(e)) return rc;
    if (!d_dst) return fail(OC_ERR_INVALID_ARG, "oc_export_states: NULL destination");
    if (int rc = check_range(e, first, count, "oc_export_states")) return rc;
    OC_ON_ENGINE_DEVICE(e);
    note_stream(e, static_cast<hipStream_t>(stream));
    OC_HIP(hipMemcpyAsync(d_dst, e->d_state + first * e->recq, static_cast<size_t>(count) * e->recq * 16, hipMemcpyDeviceToDevice,
                          static_cast<hipStream_t>(stream)));
    return OC_OK;
}

int oc_import_states(oc_engine *e, int64_t first, int64_t count, const void *d_src, void *stream) {
    if (int rc = check_engine(e)) return rc;
    if (!d_src) return fail(OC_ERR_INVALID_ARG, "oc_import_states: NULL source");
    if (int rc = check_range(e, first, count, "oc_import_states")) return rc;
    OC_ON_ENGINE_DEVICE(e);
    note_stream(e, static_cast<hipStream_t>(stream));
    OC_HIP(hipMemcpyAsync(e->d_state + first * e->recq, d_src, static_cast<size_t>(count) * e->recq * 16, hipMemcpyDeviceToDevice,
                          static_cast<hipStream_t>(stream)));
    return OC_OK;
}

static int import_checked_impl(oc_engine *e, int64_t first, int64_t count, const void *d_src, int32_t *d_rejected, void *stream, int copy,
                               const char *who) {
    if (int rc = check_engine(e)) return rc;
    if (!d_src || !d_rejected) return fail(OC_ERR_INVALID_ARG, "%s: NULL pointer", who);
    if (reinterpret_cast<uintptr_t>(d_src) % 16) return fail(OC_ERR_INVALID_ARG, "%s: records must be 16-byte aligned", who);
    if (int rc = check_range(e, first, count, who)) return rc;
    OC_ON_ENGINE_DEVICE(e);
    note_stream(e, static_cast<hipStream_t>(stream));
    hipStream_t s = static_cast<hipStream_t>(stream);
    OC_HIP(hipMemsetAsync(d_rejected, 0, sizeof(int32_t), s));
    if (count == 0) return OC_OK;
    hipLaunchKernelGGL(oc_import_checked_kernel, dim3(static_cast<unsigned>((count + 255) / 256)), dim3(256), 0, s, e->d_state + first * e->recq,
                       static_cast<const uint4 *>(d_src), count, e->recq, e->S, e->params.width, e->params.height, e->P, copy, d_rejected);
    OC_HIP(hipGetLastError());
    return OC_OK;
}

int oc_import_states_checked(oc_engine *e, int64_t first, int64_t count, const void *d_src, int32_t *d_rejected, void *stream) {
    return import_checked_impl(e, first, count, d_src, d_rejected, stream, 1, "oc_import_states_checked");
}

int oc_validate_states(oc_engine *e, int64_t count, const void *d_src, int32_t *d_rejected, void *stream) {
    return import_checked_impl(e, 0, count, d_src, d_rejected, stream, 0, "oc_validate_states");
}

int oc_prepare_kernels(oc_engine *e) {
    if (int rc = check_engine(e)) return rc;
    if (e->np_path || !e->jit.mod) return OC_OK;            // nothing is built lazily for these
    OC_ON_ENGINE_DEVICE(e);
    if (has_fresh_geometry(e)) (void)ensure_fresh_module(e, fresh_tuning(e));
    (void)ensure_fused_module(e, fused_tuning(e));
    (void)ensure_2p_module(e, own_tuning(e));
    // the module oc_encode_trajectory / oc_encode_states_batch run a small-batch engine's trajectories from (launch_observe_batch)
    if (!e->tuned_by_user && e->kpw < 16 && 16 * e->recq <= kMaxQ * kWave) (void)ensure_batch_module(e, Tuning{16, 4, kpp_for(e->S, 4)});
    return OC_OK;
}

int oc_set_tuning(oc_engine *e, int kitchens_per_wave, int passes_per_flush, int waves_per_cu) {
    if (int rc = check_engine(e)) return rc;
    if (e->np_path) {
        // the N-player kernel (oc_np_kernels.h): kitchens per group (K x players <= 64: one poke lane per player), passes per flush,
        // persistent wavefronts per CU; 0 keeps a value, and an engine never tuned chooses per launch (np_geometry)
        const int K = kitchens_per_wave ? kitchens_per_wave : (e->tuned_by_user ? e->kpw : 16);
        const int G = passes_per_flush ? passes_per_flush : (e->tuned_by_user ? e->gpasses : 2);
        const int w = waves_per_cu ? waves_per_cu : (e->tuned_by_user ? e->waves_per_cu : 8);
        if (K < 1 || K * e->P > kWave) return fail(OC_ERR_INVALID_ARG, "oc_set_tuning: kitchens_per_wave x players must be in 1..64");
        if (K * e->recq > 256) return fail(OC_ERR_INVALID_ARG, "oc_set_tuning: kitchens_per_wave %d x %d B records exceeds the 4096 B prefetch window", K, e->recq * 16);
        if (G < 1 || G > 8) return fail(OC_ERR_INVALID_ARG, "oc_set_tuning: passes_per_flush must be in 1..8");
        if (w < 1 || w > 32) return fail(OC_ERR_INVALID_ARG, "oc_set_tuning: waves_per_cu must be in 1..32");
        if (oc_np::np_lds_bytes(e->S, e->P, e->recd, oc_np::NpGeom{K, G}) > 64 * 1024) return fail(OC_ERR_INVALID_ARG, "oc_set_tuning: more than 64 KiB of LDS per wave");
        e->tuned_by_user = true;
        e->kpw = K; e->gpasses = G; e->waves_per_cu = w;
        return OC_OK;
    }
    const int kpw = kitchens_per_wave ? kitchens_per_wave : e->kpw;
    const int gp = passes_per_flush ? passes_per_flush : e->gpasses;
    const int wpc = waves_per_cu ? waves_per_cu : e->waves_per_cu;
    // a group's first byte in a viewer plane is group * kpw * S * 20: 16-byte aligned for every group iff kpw*S*5 % 4 == 0
    if (kpw < 1 || kpw > 64 || (kpw * e->S * 5) % 4)
        return fail(OC_ERR_INVALID_ARG, "oc_set_tuning: kitchens_per_wave must be in 1..64 with kitchens_per_wave * tiles a multiple of 4 (any multiple of 4 works)");
    if (kpw * e->recq > kMaxQ * kWave)
        return fail(OC_ERR_INVALID_ARG, "oc_set_tuning: kitchens_per_wave %d x %d B records exceeds the %d B prefetch window", kpw, e->recq * 16, kMaxQ * kWave * 16);
    if (gp < 1 || gp > 8) return fail(OC_ERR_INVALID_ARG, "oc_set_tuning: passes_per_flush must be in 1..8");
    if (wpc < 1 || wpc > 32) return fail(OC_ERR_INVALID_ARG, "oc_set_tuning: waves_per_cu must be in 1..32");
    if (lds_bytes(e, kpw, gp) > 64 * 1024) return fail(OC_ERR_INVALID_ARG, "oc_set_tuning: %zu B of LDS per wave exceeds 64 KiB", lds_bytes(e, kpw, gp));
    const bool rebuild = kpw != e->kpw || gp != e->gpasses || (wpc + 3) / 4 != (e->waves_per_cu + 3) / 4 || e->jit_fused.mod != nullptr || e->first_passes != 0 || e->encode_ilp4 != 0;
    e->tuned_by_user = true;
    e->first_passes = 0;                                  // (every flush of a group as long as asked for)
    e->encode_ilp4 = 0;
    e->kpw = kpw;
    e->gpasses = gp;
    e->kpp = kpp_for(e->S, gp);
    e->waves_per_cu = wpc;
    if (rebuild) {
        OC_ON_ENGINE_DEVICE(e);
        OC_HIP(hipDeviceSynchronize());          // the old module may still be executing
        jit_build(e);
    }
    return OC_OK;
}

#ifdef OC_DIAGNOSTICS
int oc_exp_set_cu_budget(oc_engine *e, int32_t cus) { return oc_internal_set_cu_budget(e, cus); }   // (experiments live in the diagnostics library only)
#endif

const char *oc_kernel_build_info(const oc_engine *e) { return e ? e->jit_status : ""; }

long long oc_debug_jit_builds(void) { return g_jit_builds; }

/* Compile-only check of the per-engine kernel build (no GPU needed): returns OC_OK and the code object
 * size, or the compiler log.  Used by the CPU test-suite and __graft_entry__.build(). */
int oc_debug_jit_compile(const oc_layout_params *p, int64_t n_kitchens, const char *arch, int64_t *code_bytes,
                         char *log_out, int64_t log_cap) {
    if (!p || !arch) return fail(OC_ERR_INVALID_ARG, "oc_debug_jit_compile: NULL argument");
    oc_engine tmp = oc_engine();
    std::vector<uint32_t> tabs;
    if (int rc = prepare_engine(p, n_kitchens, &tmp, tabs)) return rc;
    std::vector<char> code;
    std::string log;
    if (const char *tn = OC_DIAG_ENV("OC_DEBUG_TUNING")) {             // diagnostics: "kpw,passes,waves per CU" of the build under test
        int k = 0, g = 0, w = 0;
        if (sscanf(tn, "%d,%d,%d", &k, &g, &w) == 3 && k > 0 && g > 0 && w > 0) { tmp.kpw = k; tmp.gpasses = g; tmp.waves_per_cu = w; tmp.kpp = kpp_for(tmp.S, g); }
    }
    const char *dump = OC_DIAG_ENV("OC_DEBUG_DUMP_CODE");               // diagnostics: the code object to this file
    const char *fresh = OC_DIAG_ENV("OC_DEBUG_FRESH");                  // diagnostics: the module for fresh destinations instead
    const int rc = jit_compile_text((fresh && fresh[0] == '1') ? jit_source_single(&tmp, Tuning{16, 4, kpp_for(tmp.S, 4), tmp.S > 32 ? 1 : 2}, SRC_FRESH, kFreshWavesPerCu)
                                                               : jit_source_single(&tmp), arch, code, log);
    if (rc == OC_OK && dump) { if (FILE *f = fopen(dump, "wb")) { fwrite(code.data(), 1, code.size(), f); fclose(f); } }
    if (code_bytes) *code_bytes = static_cast<int64_t>(code.size());
    if (log_out && log_cap > 0) snprintf(log_out, static_cast<size_t>(log_cap), "%s", log.c_str());
    if (rc != OC_OK) return fail(rc, "hiprtc compile failed: %.400s", log.c_str());
    return OC_OK;
}

/* Ahead-of-time build (no GPU needed; __graft_entry__.build()): every module an engine of this shape loads -- oc_create's, the one for
 * fresh (time-major) destinations, the K-steps-per-launch rollout's, the batched featurisation's -- compiled for `arch` as the device
 * reports it ("gfx950:sramecc+:xnack-") and written to out_dir/<hash>.hsaco.  *n_modules (optional): how many. */
int oc_debug_aot_build(const oc_layout_params *p, int64_t n_kitchens, const char *arch, const char *out_dir, int32_t *n_modules) {
    if (!p || !arch || !out_dir || !out_dir[0]) return fail(OC_ERR_INVALID_ARG, "oc_debug_aot_build: NULL argument");
    oc_engine tmp = oc_engine();
    std::vector<uint32_t> tabs;
    if (int rc = prepare_engine(p, n_kitchens, &tmp, tabs)) return rc;
    if (n_modules) *n_modules = 0;
    if (tmp.np_path) return OC_OK;                                    // (the N-player kernels are part of the library itself)
    snprintf(tmp.arch, sizeof(tmp.arch), "%s", arch);
    (void)mkdir(out_dir, 0755);
    std::vector<std::string> texts;
    texts.push_back(jit_source_single(&tmp));
    if (fresh_geometry_shape(&tmp)) texts.push_back(jit_source_single(&tmp, fresh_tuning_shape(&tmp), SRC_FRESH, kFreshWavesPerCu));
    texts.push_back(jit_source_single(&tmp, fused_tuning(&tmp), SRC_ROLLOUT, tmp.waves_per_cu));
    texts.push_back(jit_source_single(&tmp, own_tuning(&tmp), SRC_TWOPTR, tmp.waves_per_cu));
    if (tmp.kpw < 16 && 16 * tmp.recq <= kMaxQ * kWave) texts.push_back(jit_source_single(&tmp, Tuning{16, 4, kpp_for(tmp.S, 4)}, SRC_BATCH, kFreshWavesPerCu));
    g_aot_out = out_dir;
    int rc = OC_OK;
    std::string log;
    for (const std::string &t : texts) {
        std::vector<char> code;
        rc = jit_compile_text(t, arch, code, log);
        if (rc != OC_OK) break;
        if (n_modules) ++*n_modules;
    }
    g_aot_out.clear();
    if (rc != OC_OK) return fail(rc, "oc_debug_aot_build: hiprtc compile failed: %.400s", log.c_str());
    return OC_OK;
}

/* The same for a group module (one launch over n_engines engines): plans the geometry for `num_cus` CUs and compiles.
 * plan_out (optional, 2 * n_engines ints): kitchens per wavefront group and blocks of every engine. */
int oc_debug_jit_compile_group(const oc_layout_params *params, const int64_t *n_kitchens, int32_t n_engines, int32_t num_cus, const char *arch,
                               int64_t *code_bytes, int32_t *plan_out, char *log_out, int64_t log_cap) {
    if (!params || !n_kitchens || !arch || n_engines < 1 || n_engines > kMaxSegments)
        return fail(OC_ERR_INVALID_ARG, "oc_debug_jit_compile_group: bad argument");
    std::vector<oc_engine> tmp(n_engines);
    oc_group g;
    g.mod = nullptr;
    for (int i = 0; i < n_engines; ++i) {
        std::vector<uint32_t> tabs;
        if (int rc = prepare_engine(&params[i], n_kitchens[i], &tmp[i], tabs)) return rc;
        g.engines.push_back(&tmp[i]);
    }
    g.device = -1;
    g.waves_per_cu = 12;
    g.num_cus = num_cus > 0 ? num_cus : 256;
    if (int rc = group_plan(&g, nullptr, 0, 0)) return rc;
    std::vector<const oc_engine *> es(g.engines.begin(), g.engines.end());
    std::vector<char> code;
    std::string log;
    const int rc = jit_compile_text(jit_source_group(es, g.tunings, (g.waves_per_cu + 3) / 4, g.layout_of_seg), arch, code, log);
    if (code_bytes) *code_bytes = static_cast<int64_t>(code.size());
    if (plan_out)
        for (int i = 0; i < n_engines; ++i) { plan_out[2 * i] = g.tunings[i].kpw; plan_out[2 * i + 1] = g.blocks[i]; }
    if (log_out && log_cap > 0) snprintf(log_out, static_cast<size_t>(log_cap), "%s", log.c_str());
    if (rc != OC_OK) return fail(rc, "hiprtc compile failed: %.400s", log.c_str());
    return OC_OK;
}

/* ... and written to out_dir like oc_debug_aot_build does (the group module of oc_group_create for these engines, in this order). */
int oc_debug_aot_build_group(const oc_layout_params *params, const int64_t *n_kitchens, int32_t n_engines, int32_t num_cus, const char *arch,
                             const char *out_dir) {
    if (!out_dir || !out_dir[0]) return fail(OC_ERR_INVALID_ARG, "oc_debug_aot_build_group: NULL out_dir");
    (void)mkdir(out_dir, 0755);
    g_aot_out = out_dir;
    const int rc = oc_debug_jit_compile_group(params, n_kitchens, n_engines, num_cus, arch, nullptr, nullptr, nullptr, 0);
    g_aot_out.clear();
    return rc;
}

#ifdef OC_DIAGNOSTICS
/* Diagnostics build (overcooked_debug.h): per-wave phase timestamps of the next launches. */
int oc_debug_trace(oc_engine *e, int enable, unsigned long long *host_out, int64_t max_waves) {
    if (int rc = check_engine(e)) return rc;
    const int64_t cap = 32 * 1024;
    OC_ON_ENGINE_DEVICE(e);
    if (enable) {
        if (!e->d_trace) OC_HIP(hipMalloc(reinterpret_cast<void **>(&e->d_trace), cap * 16 * sizeof(unsigned long long)));
        OC_HIP(hipMemset(e->d_trace, 0, cap * 16 * sizeof(unsigned long long)));
        return OC_OK;
    }
    if (host_out && e->d_trace) {
        OC_HIP(hipDeviceSynchronize());
        OC_HIP(hipMemcpy(host_out, e->d_trace, static_cast<size_t>(max_waves < cap ? max_waves : cap) * 16 * sizeof(unsigned long long), hipMemcpyDeviceToHost));
    }
    if (e->d_trace) { (void)hipFree(e->d_trace); e->d_trace = nullptr; }
    return OC_OK;
}
#endif  // OC_DIAGNOSTICS

}  // extern "C"
