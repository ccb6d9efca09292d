// Between the head's logits and the choice of a token: the penalties for repeated tokens, a
// bias and a grammar mask, one pass over the logits (bf16, fp16, fp32).
//
// For row b and token v, with the row's history h[b, 0 .. len_b) of which the first prompt_b
// entries are the prompt:
//   seen  = v occurs in the history; n = how often it occurs after the prompt
//   x = logits[b, v]
//   x = x > 0 ? x / repetition_b : x * repetition_b     where seen
//   x = x - frequency_b n - presence_b [n > 0]
//   x = x + bias[v];   x = -inf where the mask's bit is 0
// in fp32, rounded once.
//
// A workgroup takes a slice of one row's vocabulary.  The slice's counts are a table in LDS
// (bit 31: seen in the prompt, the rest: n) that the workgroup fills by scanning the row's
// history -- integer LDS atomics, so the order does not matter -- and the logits then stream
// past it.  The scan is repeated by every slice of the row, so slices are as long as the
// grid allows up to 8192 tokens (longer ones leave fewer waves to hide the loads: 81 us at 8192,
// 86 at 16384 for 256 x 131072; the rule is at the launch).  Bound by HBM at large batches (the
// logits read and written once, the bias once, a bit of mask a token: 256 x 131072 fp32 with
// all of them and 4096-token histories 76 us, 5.4 TB/s).
#include "../../include/nsmoe.h"
#include "gemm_core.h"
#include "nsmoe_capi_internal.h"

namespace nsmoe {

constexpr int LG_NT = 512;
constexpr int LG_VEC = 8;           // logits per thread and step: one byte of mask
constexpr int LG_MAX_SLICE = 8192;   // 32 KiB of table: four workgroups per CU
constexpr int LG_MIN_SLICE = 1024;
constexpr int LG_IDS = 8;            // history loads of a thread in flight

struct LogitParams {
  const void* x;
  void* y;
  int64_t ldx, ldy;
  const int64_t* hist;
  int64_t ldh, L;
  const int32_t* lens;
  const int32_t* prompt;
  const float *rep, *freq, *pres;
  const float* bias;
  int64_t ldb;
  const uint8_t* mask;
  int64_t ldm;  // bytes
  int V, slice;
};

// 8 elements from any element-aligned address: the vectors of a row whose length is odd do
// not start at 16 bytes, and gfx950 loads and stores them all the same.
template <class T>
struct __attribute__((packed, aligned(sizeof(T)))) Run8 { T e[LG_VEC]; };

template <int DT, int ODT, bool HIST>
__global__ void __launch_bounds__(LG_NT) logits_kernel(LogitParams p) {
  using TI = typename Elem<DT>::T;
  using TO = typename Elem<ODT>::T;
  extern __shared__ __attribute__((aligned(16))) uint32_t s_tab[];
  const int64_t b = blockIdx.y;
  const int v0 = (int)blockIdx.x * p.slice;
  const int nv = min(p.slice, p.V - v0);
  const int tid = threadIdx.x;

  if constexpr (HIST) {
    for (int i = tid * 4; i < p.slice; i += LG_NT * 4) *(u32x4*)(s_tab + i) = u32x4{0, 0, 0, 0};
    __syncthreads();
    int64_t n = p.lens ? p.lens[b] : p.L;
    n = n < 0 ? 0 : n > p.L ? p.L : n;
    const int64_t np = p.prompt ? p.prompt[b] : 0;
    const int64_t* h = p.hist + b * p.ldh;
    for (int64_t j0 = tid; j0 < n; j0 += LG_IDS * LG_NT) {
      int64_t id[LG_IDS];
#pragma unroll
      for (int u = 0; u < LG_IDS; ++u) {
        const int64_t j = j0 + u * LG_NT;
        id[u] = j < n ? h[j] : -1;
      }
#pragma unroll
      for (int u = 0; u < LG_IDS; ++u) {
        const uint64_t at = (uint64_t)id[u] - (uint64_t)v0;
        if (id[u] < 0 || at >= (uint64_t)nv) continue;
        if (j0 + u * LG_NT < np) atomicOr(&s_tab[at], 0x80000000u);
        else atomicAdd(&s_tab[at], 1u);
      }
    }
    __syncthreads();
  }
  const float rep = HIST && p.rep ? p.rep[b] : 1.0f;
  const float freq = HIST && p.freq ? p.freq[b] : 0.0f;
  const float pres = HIST && p.pres ? p.pres[b] : 0.0f;
  const TI* x = (const TI*)p.x + b * p.ldx + v0;
  TO* y = (TO*)p.y + b * p.ldy + v0;
  const float* bias = p.bias ? p.bias + b * p.ldb + v0 : nullptr;
  const uint8_t* mask = p.mask ? p.mask + b * p.ldm + v0 / 8 : nullptr;

  auto change = [&](float v, uint32_t word, float bv, bool allowed) {
    if constexpr (HIST) {
      if (word) {
        v = v > 0.0f ? v / rep : v * rep;
        const uint32_t n = word & 0x7fffffffu;
        if (n) v = v - freq * (float)n - pres;
      }
    }
    v += bv;
    return allowed ? v : -INFINITY;
  };
  // Two steps' loads are issued before the first one's store, which may be to the same memory
  // and holds later loads back.
  constexpr int U = 2;
  for (int i0 = tid * LG_VEC; i0 < nv; i0 += U * LG_NT * LG_VEC) {
    Run8<TI> in[U];
    Run8<float> bv[U] = {};
    uint32_t bits[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int i = i0 + k * LG_NT * LG_VEC;
      bits[k] = mask && i < nv ? mask[i / 8] : 0xffu;
      if (i + LG_VEC <= nv) {
        in[k] = *(const Run8<TI>*)(x + i);
        if (bias) bv[k] = *(const Run8<float>*)(bias + i);
      }
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int i = i0 + k * LG_NT * LG_VEC;
      if (i >= nv) break;
      uint32_t w[LG_VEC] = {};
      if constexpr (HIST) {
        const u32x4 a = *(const u32x4*)(s_tab + i), c = *(const u32x4*)(s_tab + i + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = a[e], w[4 + e] = c[e];
      }
      if (i + LG_VEC <= nv) {
        float o[LG_VEC];
#pragma unroll
        for (int e = 0; e < LG_VEC; ++e)
          o[e] = change(Elem<DT>::to_f(in[k].e[e]), w[e], bv[k].e[e], (bits[k] >> e) & 1);
        TO r[LG_VEC];
        round_to<ODT>(o, r);
        Run8<TO> out;
#pragma unroll
        for (int e = 0; e < LG_VEC; ++e) out.e[e] = r[e];
        *(Run8<TO>*)(y + i) = out;
      } else {
#pragma unroll
        for (int e = 0; e < LG_VEC; ++e)
          if (i + e < nv)
            y[i + e] = Elem<ODT>::from_f(change(Elem<DT>::to_f(x[i + e]), w[e],
                                                bias ? bias[i + e] : 0.0f, (bits[k] >> e) & 1));
      }
    }
  }
}

template <int DT, int ODT>
static int logits_launch(const LogitParams& P, dim3 grid, hipStream_t s) {
  KernelTimer timer("logits", s);
  if (P.hist)
    logits_kernel<DT, ODT, true><<<grid, LG_NT, (size_t)P.slice * 4, s>>>(P);
  else
    logits_kernel<DT, ODT, false><<<grid, LG_NT, 0, s>>>(P);
  timer.stop();
  return check_launch("logits_kernel");
}

}  // namespace nsmoe

using namespace nsmoe;

extern "C" int nsmoe_penalize_logits(const nsmoe_logits_args* a, void* stream) {
  NSMOE_REQUIRE(a, "penalize_logits: NULL args");
  NSMOE_REQUIRE(a->dtype >= DT_BF16 && a->dtype <= DT_F32 &&
                    (a->out_dtype == a->dtype || a->out_dtype == DT_F32),
                "penalize_logits: dtype %d to %d (the same type, or fp32 out)", a->dtype,
                a->out_dtype);
  NSMOE_REQUIRE(a->batch >= 0 && a->batch <= 65535, "penalize_logits: batch %lld (at most 65535)",
                (long long)a->batch);
  NSMOE_REQUIRE(a->vocab >= 0 && a->vocab < (1 << 30), "penalize_logits: bad vocab %d", a->vocab);
  NSMOE_REQUIRE(a->history_cap >= 0 && a->history_cap < INT32_MAX,
                "penalize_logits: bad history length");
  if (a->batch == 0 || a->vocab == 0) return NSMOE_OK;
  NSMOE_REQUIRE(a->logits && a->out && (a->history || a->history_cap == 0),
                "penalize_logits: NULL pointer");
  const int es = a->dtype == DT_F32 ? 4 : 2, eo = a->out_dtype == DT_F32 ? 4 : 2;
  NSMOE_REQUIRE(((uintptr_t)a->logits & (es - 1)) == 0 && ((uintptr_t)a->out & (eo - 1)) == 0 &&
                    ((uintptr_t)a->bias & 3) == 0 && ((uintptr_t)a->history & 7) == 0,
                "penalize_logits: misaligned pointer");
  LogitParams P{};
  P.x = a->logits;
  P.y = a->out;
  P.ldx = a->logits_stride;
  P.ldy = a->out_stride;
  const bool hist = a->history_cap > 0 && (a->repetition || a->frequency || a->presence);
  P.hist = hist ? a->history : nullptr;
  P.ldh = a->history_stride;
  P.L = a->history_cap;
  P.lens = a->lens;
  P.prompt = a->prompt_lens;
  P.rep = a->repetition;
  P.freq = a->frequency;
  P.pres = a->presence;
  P.bias = a->bias;
  P.ldb = a->bias_stride;
  P.mask = (const uint8_t*)a->mask;
  P.ldm = a->mask_stride * 4;
  P.V = a->vocab;
  // Slices of 1024 to 8192 tokens, whole 64s: two workgroups a CU over the batch.
  const int64_t want = cdiv(2 * device_cus(), a->batch);  // slices per row
  int64_t slice = cdiv(cdiv(a->vocab, want), 64) * 64;
  slice = slice < LG_MIN_SLICE ? LG_MIN_SLICE : slice > LG_MAX_SLICE ? LG_MAX_SLICE : slice;
  P.slice = (int)slice;
  const dim3 grid((unsigned)cdiv(a->vocab, slice), (unsigned)a->batch);
  hipStream_t s = (hipStream_t)stream;
  if (a->dtype == DT_F32) return logits_launch<DT_F32, DT_F32>(P, grid, s);
  if (a->dtype == DT_BF16)
    return a->out_dtype == DT_F32 ? logits_launch<DT_BF16, DT_F32>(P, grid, s)
                                  : logits_launch<DT_BF16, DT_BF16>(P, grid, s);
  return a->out_dtype == DT_F32 ? logits_launch<DT_F16, DT_F32>(P, grid, s)
                                : logits_launch<DT_F16, DT_F16>(P, grid, s);
}
