// Eviction from a key/value cache by accumulated attention weight.
//
// For a sequence b with n = lens[b] cached rows and a budget of m: where n <= m every row is
// kept; otherwise the first `sinks` rows, the last `recent` and, of those between, the
// r = m - sinks - recent with the largest weights w[b, h, .] (ties: the lower index), chosen
// for each key/value head h on its own.  Kept rows move to the front in index order.
//
//   evict_select_kernel  one workgroup per (sequence, head): the r-th largest weight by a
//                        radix descent over order-preserving 32-bit keys (histograms of 11, 11
//                        and 10 bits in LDS), then one ordered pass that writes the kept
//                        indices, weights and the new length.  Each wave owns a contiguous
//                        run of the row, so an index's place is the counts of the waves
//                        before it plus a ballot within the wave.  Up to 8192 rows the weights
//                        are read once and stay in registers (8 a lane) over the passes;
//                        longer rows are read again each pass, from L2.
//   evict_move_kernel    copies the kept key and value rows, 16 bytes a thread, by those
//                        indices.
//
// The move reads and writes the kept rows once, which is nearly all of the traffic: bound by
// HBM at large caches (32 x 8192 rows down to 2048, 8 heads of 128: 14 us and 100 us, the move
// at 5 TB/s), by the selection's chain of passes at small ones (8 x 1100 rows: 10 us and 4).
//
// Weights order as floats with -0 equal to +0; a NaN counts as the largest (it is kept, where
// it can be seen, rather than lost).
#include "../../include/nsmoe.h"
#include "gemm_core.h"
#include "nsmoe_capi_internal.h"

namespace nsmoe {

constexpr int EV_NT = 1024;
constexpr int EV_WAVES = EV_NT / 64;
constexpr int EV_BINS = 2048;
constexpr int EV_HOLD = 8;  // weights of a lane in registers
constexpr int EV_MOVE_NT = 256;

struct EvictParams {
  const char *k, *v;
  char *k_out, *v_out;
  int64_t ksb, kst, ksh, vsb, vst, vsh;        // bytes: batch, row, head
  int64_t kob, kot, koh, vob, vot, voh;
  const float* w;
  float* w_out;
  int64_t wsb, wsh, wob, woh;                  // elements: batch, head
  const int32_t* lens;
  int32_t* lens_out;
  int32_t* index;                              // [B, H, m]
  int64_t S, So;                               // rows of the cache and of the output
  int B, H, m, recent, sinks, row_bytes, zero_tail, stream;
};

// Keys whose unsigned order is the weights' order: NaN above everything, -0 as +0.
__device__ __forceinline__ uint32_t evict_key(float f) {
  if (f != f) return 0xffffffffu;
  const uint32_t u = __float_as_uint(f + 0.0f);  // -0 + 0 = +0
  return (u >> 31) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int evict_len(const EvictParams& p, int b) {
  const int64_t n = p.lens[b];
  return (int)(n < 0 ? 0 : n > p.S ? p.S : n);
}

__global__ void __launch_bounds__(EV_NT) evict_select_kernel(EvictParams p) {
  __shared__ uint32_t s_hist[EV_BINS];
  __shared__ __attribute__((aligned(16))) uint32_t s_wave[EV_WAVES], s_wave2[EV_WAVES];
  __shared__ uint32_t s_bin, s_left;
  const int b = blockIdx.x / p.H, h = blockIdx.x % p.H;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = evict_len(p, b), m = p.m;
  const float* w = p.w + b * p.wsb + h * p.wsh;
  float* wo = p.w_out + b * p.wob + h * p.woh;
  int32_t* idx = p.index + (int64_t)blockIdx.x * m;
  const int kept = n < m ? n : m;
  if (h == 0 && tid == 0) p.lens_out[b] = kept;
  // Behind the kept rows: no index, and the weights of a buffer of our own are zero.
  for (int i = kept + tid; i < m; i += EV_NT) idx[i] = -1;
  if (p.zero_tail)
    for (int64_t i = kept + tid; i < p.So; i += EV_NT) wo[i] = 0.0f;
  if (n <= m) {
    for (int i = tid; i < n; i += EV_NT) {
      idx[i] = i;
      wo[i] = w[i];
    }
    return;
  }
  const int lo = p.sinks, hi = n - p.recent;  // the rows that compete
  // The wave's run of [0, n): whole steps of 64, in turns of EV_HOLD steps.
  const int steps = ((n + EV_WAVES - 1) / EV_WAVES + 63) / 64;
  const int w0 = wave * steps * 64, w1 = min(n, w0 + steps * 64);
  const int turns = (steps + EV_HOLD - 1) / EV_HOLD;
  float f[EV_HOLD];
  auto load = [&](int turn) {
#pragma unroll
    for (int u = 0; u < EV_HOLD; ++u) {
      const int i = w0 + (turn * EV_HOLD + u) * 64 + lane;
      f[u] = i < w1 ? w[i] : 0.0f;
    }
  };
  // each(row, weight) over the wave's rows, 64 lanes a step (past the run's end: row >= w1)
  auto sweep = [&](auto&& each) {
    for (int turn = 0; turn < turns; ++turn) {
      if (turns > 1) load(turn);
#pragma unroll
      for (int u = 0; u < EV_HOLD; ++u)
        if (turn * EV_HOLD + u < steps) each(w0 + (turn * EV_HOLD + u) * 64 + lane, f[u]);
    }
  };
  if (turns == 1) load(0);
  uint32_t left = (uint32_t)(m - p.sinks - p.recent);
  // The descent: `prefix` holds the decided high bits of the threshold key, `left` how many
  // keys are still to be taken among those that share it.  left == 0 takes none: any
  // threshold above every key would do, and the top one with no ties taken is such.
  uint32_t prefix = 0, mask = 0;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int sh = pass == 0 ? 21 : pass == 1 ? 10 : 0, nb = pass == 2 ? 1024 : 2048;
    for (int i = tid; i < nb; i += EV_NT) s_hist[i] = 0;
    __syncthreads();
    sweep([&](int i, float x) {
      const uint32_t key = evict_key(x);
      if (i >= lo && i < hi && i < w1 && (key & mask) == prefix)
        atomicAdd(&s_hist[(key >> sh) & (nb - 1)], 1u);
    });
    __syncthreads();
    // The bin, from the top, in which the running count reaches `left`: thread t holds two
    // bins (the second histogram half is empty for 10 bits).
    const int b1 = nb - 1 - 2 * tid, b0 = b1 - 1;
    const uint32_t c1 = b1 >= 0 ? s_hist[b1] : 0, c0 = b0 >= 0 ? s_hist[b0] : 0;
    const uint32_t incl = (uint32_t)wave_scan_incl((int)(c1 + c0));
    if (lane == 63) s_wave[wave] = incl;
    __syncthreads();
    uint32_t before = incl - c1 - c0;
#pragma unroll
    for (int k = 0; k < EV_WAVES; ++k) before += k < wave ? s_wave[k] : 0;
    // exactly one thread holds the bin that `left` falls into (left >= 1)
    if (left > before && left <= before + c1) {
      s_bin = (uint32_t)b1;
      s_left = left - before;
    } else if (left > before + c1 && left <= before + c1 + c0) {
      s_bin = (uint32_t)b0;
      s_left = left - before - c1;
    }
    __syncthreads();
    if (left) {
      left = s_left;
      prefix |= s_bin << sh;
    } else {
      prefix |= (uint32_t)(nb - 1) << sh;
    }
    mask |= (uint32_t)(nb - 1) << sh;
    __syncthreads();
  }
  // Keys above `prefix` are kept, of those equal to it the first `left`.  With nothing to
  // take, prefix is 0xffffffff: no key is above it, and left is 0.

  // Each wave counts, then writes, its own run.
  uint32_t above = 0, equal = 0;  // this lane's
  sweep([&](int i, float x) {
    const bool live = i < w1, held = i < lo || i >= hi;
    const uint32_t key = evict_key(x);
    above += live && (held || key > prefix);
    equal += live && !held && key == prefix;
  });
  for (int o = 32; o; o >>= 1) above += __shfl_xor(above, o), equal += __shfl_xor(equal, o);
  if (lane == 0) s_wave[wave] = above, s_wave2[wave] = equal;
  __syncthreads();
  uint32_t at = 0, ties = 0;  // kept, and ties met, before this wave's run
#pragma unroll
  for (int k = 0; k < EV_WAVES; ++k) {
    at += k < wave ? s_wave[k] : 0;
    ties += k < wave ? s_wave2[k] : 0;
  }
  at += ties < left ? ties : left;
  sweep([&](int i, float x) {
    const bool live = i < w1, held = live && (i < lo || i >= hi);
    const uint32_t key = evict_key(x);
    const bool tie = live && !held && key == prefix;
    const uint64_t tb = __ballot(tie), below = ((uint64_t)1 << lane) - 1;
    const bool take = held || (live && !held && key > prefix) ||
                      (tie && ties + (uint32_t)__popcll(tb & below) < left);
    const uint64_t kb = __ballot(take);
    if (take) {
      const uint32_t o = at + (uint32_t)__popcll(kb & below);
      idx[o] = i;
      wo[o] = x;
    }
    at += (uint32_t)__popcll(kb);
    ties += (uint32_t)__popcll(tb);
  });
}

// One thread per 16 bytes (or 2 bytes, where rows are not aligned) of a row of the output in
// order, so a wave writes neighbouring addresses; a workgroup takes EV_MOVE_STEPS turns.
constexpr int EV_MOVE_STEPS = 2;

template <class T>
__global__ void __launch_bounds__(EV_MOVE_NT) evict_move_kernel(EvictParams p, LaunchDiv by_row,
                                                                LaunchDiv by_heads, int rows) {
  const int b = blockIdx.y;
  const uint32_t items = (uint32_t)rows * by_heads.d * by_row.d;
  const char *k = p.k + b * p.ksb, *v = p.v + b * p.vsb;
  char *ko = p.k_out + b * p.kob, *vo = p.v_out + b * p.vob;
  const uint32_t it0 = blockIdx.x * (EV_MOVE_NT * EV_MOVE_STEPS) + threadIdx.x;
  int src[EV_MOVE_STEPS];
  uint32_t r[EV_MOVE_STEPS], c[EV_MOVE_STEPS];
#pragma unroll
  for (int u = 0; u < EV_MOVE_STEPS; ++u) {
    const uint32_t it = it0 + u * EV_MOVE_NT;
    r[u] = by_row.div(it);
    c[u] = it - r[u] * by_row.d;
    const uint32_t o = by_heads.div(r[u]), h = r[u] - o * by_heads.d;
    src[u] = -1;
    if (it < items && o < (uint32_t)p.m) src[u] = p.index[((int64_t)b * p.H + h) * p.m + o];
  }
  T kv[EV_MOVE_STEPS], vv[EV_MOVE_STEPS];
#pragma unroll
  for (int u = 0; u < EV_MOVE_STEPS; ++u) {
    const uint32_t o = by_heads.div(r[u]), h = r[u] - o * by_heads.d;
    const int64_t at = c[u] * (int64_t)sizeof(T);
    kv[u] = vv[u] = T{};
    if (src[u] >= 0) {
      kv[u] = *(const T*)(k + src[u] * p.kst + h * p.ksh + at);
      vv[u] = *(const T*)(v + src[u] * p.vst + h * p.vsh + at);
    }
  }
#pragma unroll
  for (int u = 0; u < EV_MOVE_STEPS; ++u) {
    const uint32_t o = by_heads.div(r[u]), h = r[u] - o * by_heads.d;
    if (it0 + u * EV_MOVE_NT >= items || (src[u] < 0 && !p.zero_tail)) continue;
    const int64_t at = c[u] * (int64_t)sizeof(T);
    T *kd = (T*)(ko + o * p.kot + h * p.koh + at), *vd = (T*)(vo + o * p.vot + h * p.voh + at);
    if (p.stream) {
      __builtin_nontemporal_store(kv[u], kd);
      __builtin_nontemporal_store(vv[u], vd);
    } else {
      *kd = kv[u];
      *vd = vv[u];
    }
  }
}

}  // namespace nsmoe

using namespace nsmoe;

extern "C" int nsmoe_cache_evict(const nsmoe_evict_args* a, void* stream) {
  NSMOE_REQUIRE(a, "cache_evict: NULL args");
  NSMOE_REQUIRE(a->elem_bytes == 2 || a->elem_bytes == 4, "cache_evict: elements of %d bytes",
                a->elem_bytes);
  NSMOE_REQUIRE(a->batch >= 0 && a->n_kv_heads >= 1 && a->head_dim >= 1 && a->head_dim <= 4096 &&
                    a->n_kv_heads <= 4096 && a->batch * a->n_kv_heads < (1 << 24),
                "cache_evict: bad batch, heads or head_dim");
  NSMOE_REQUIRE(a->cap >= 0 && a->cap < (1 << 30) && a->out_cap >= 0 && a->out_cap < (1 << 30),
                "cache_evict: bad capacity");
  NSMOE_REQUIRE(a->batch <= 65535 && a->out_cap * a->n_kv_heads * a->head_dim < (1ll << 31) - 4096,
                "cache_evict: batch %lld (at most 65535) or a sequence's output (2^31 elements) "
                "too large", (long long)a->batch);
  NSMOE_REQUIRE(a->budget >= 1 && a->budget <= a->out_cap,
                "cache_evict: budget %lld outside 1 .. the output's %lld rows",
                (long long)a->budget, (long long)a->out_cap);
  NSMOE_REQUIRE(a->recent >= 0 && a->sinks >= 0 && a->recent + a->sinks <= a->budget,
                "cache_evict: sinks %lld + recent %lld exceed the budget %lld",
                (long long)a->sinks, (long long)a->recent, (long long)a->budget);
  if (a->batch == 0) return NSMOE_OK;
  NSMOE_REQUIRE(a->lens && a->index && a->lens_out && a->weights_out && a->k_out && a->v_out &&
                    (a->cap == 0 || (a->k && a->v && a->weights)),
                "cache_evict: NULL pointer");
  NSMOE_REQUIRE(((uintptr_t)a->weights & 3) == 0 && ((uintptr_t)a->weights_out & 3) == 0,
                "cache_evict: misaligned weights");
  const int64_t es = a->elem_bytes;
  EvictParams P{};
  uint64_t bits = (uint64_t)a->k | (uint64_t)a->v | (uint64_t)a->k_out | (uint64_t)a->v_out |
                  (uint64_t)(a->head_dim * es);
  // The stride of a dim of one element may be anything.
  auto stride = [&](const int64_t* st, int64_t rows, int64_t& sb, int64_t& sr, int64_t& sh) {
    sb = a->batch > 1 ? st[0] * es : 0;
    sr = rows > 1 ? st[1] * es : 0;
    sh = a->n_kv_heads > 1 ? st[2] * es : 0;
    bits |= (uint64_t)sb | (uint64_t)sr | (uint64_t)sh;
  };
  stride(a->k_stride, a->cap, P.ksb, P.kst, P.ksh);
  stride(a->v_stride, a->cap, P.vsb, P.vst, P.vsh);
  stride(a->k_out_stride, a->out_cap, P.kob, P.kot, P.koh);
  stride(a->v_out_stride, a->out_cap, P.vob, P.vot, P.voh);
  NSMOE_REQUIRE((bits & (es - 1)) == 0, "cache_evict: misaligned pointer");
  P.k = (const char*)a->k;
  P.v = (const char*)a->v;
  P.k_out = (char*)a->k_out;
  P.v_out = (char*)a->v_out;
  P.w = a->weights;
  P.w_out = a->weights_out;
  P.wsb = a->weights_stride[0];
  P.wsh = a->weights_stride[1];
  P.wob = a->weights_out_stride[0];
  P.woh = a->weights_out_stride[1];
  P.lens = a->lens;
  P.lens_out = a->lens_out;
  P.index = a->index;
  P.S = a->cap;
  P.So = a->out_cap;
  P.B = (int)a->batch;
  P.H = a->n_kv_heads;
  P.m = (int)a->budget;
  P.recent = (int)a->recent;
  P.sinks = (int)a->sinks;
  P.row_bytes = (int)(a->head_dim * es);
  P.zero_tail = a->zero_tail != 0;
  hipStream_t s = (hipStream_t)stream;
  {
    KernelTimer timer("evict_select", s);
    evict_select_kernel<<<(unsigned)(P.B * P.H), EV_NT, 0, s>>>(P);
    timer.stop();
  }
  NSMOE_TRY(check_launch("evict_select_kernel"));
  const int rows = P.zero_tail ? (int)P.So : P.m;
  const bool vec = (bits & 15) == 0;
  const LaunchDiv by_row = launch_div(P.row_bytes / (vec ? 16 : 2)), by_heads = launch_div(P.H);
  const dim3 grid((unsigned)cdiv((int64_t)rows * P.H * by_row.d, EV_MOVE_NT * EV_MOVE_STEPS),
                  (unsigned)P.B);
  // Outputs that the 256 MiB memory-side cache cannot hold beside what is read are stored past
  // it (32 x 2048 kept rows of 8 heads of 128: 116 us against 121 for the whole call).
  P.stream = 4 * (int64_t)P.B * rows * P.H * P.row_bytes > (256ll << 20);
  KernelTimer timer("evict_move", s);
  if (vec) evict_move_kernel<u32x4><<<grid, EV_MOVE_NT, 0, s>>>(P, by_row, by_heads, rows);
  else evict_move_kernel<uint16_t><<<grid, EV_MOVE_NT, 0, s>>>(P, by_row, by_heads, rows);
  timer.stop();
  return check_launch("evict_move_kernel");
}
