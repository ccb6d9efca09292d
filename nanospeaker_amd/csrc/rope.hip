// Rotary positions of query and key heads, forward and backward (bf16, fp16, fp32).
//
// Plane j of a head turns by t = position * freq[j] (reference: src/model/rope.py):
//   y1 = a (x1 cos t - x2 sin t),   y2 = a (x2 cos t + x1 sin t)
// with x1, x2 dims (j, j + rot / 2) of the head ("rotate half") or (2 j, 2 j + 1)
// (interleaved), j < rot / 2; dims from rot on pass through.  The frequencies (with whatever
// stretch a long context asks for folded in) and the amplitude a are the caller's.  The
// backward is the same kernel with the angle negated: the rotation's transpose.
//
// A position may be far (10^6 and more), where an fp32 product position * freq has lost the
// angle: the product is formed in fp64 in turns, reduced to [-1/2, 1/2] and only then rounded
// to fp32 (2^-26 of a turn at most), and sin / cos are the library's sincospi.  The rotation
// itself is fp32 on the widened elements, rounded once to the type.
//
// A workgroup takes `tok` consecutive tokens: its threads first make the tok x rot / 2 cosines
// and sines once, into LDS (they are shared by every head of the token), then stream the
// heads of q and k, VP planes a thread and step in 16-byte vectors.  Bound by HBM at long calls
// (each element read once and written once: 4 x 8192 tokens of 9 + 3 heads of 64, bf16, 17.8 us
// or 5.6 TB/s out of a warm memory-side cache; 4 x 2047 of 32 + 8 heads of 128, fp32, 67 us or
// 5.0 TB/s) and by launch latency at decode ones (64 tokens: 3.3 us).
#include "../../include/nsmoe.h"
#include "gemm_core.h"
#include "nsmoe_capi_internal.h"

namespace nsmoe {

constexpr int RP_NT = 256;
constexpr int RP_BATCH = 4;         // items of a thread in flight
constexpr int RP_MAX_TOK = 16;      // tokens per workgroup
constexpr int RP_MAX_TRIG = 1024;   // planes x tokens held in LDS, 8 bytes each

struct RopeTensor {
  const char* src;
  char* dst;
  int64_t sb, st, sh;  // input strides in bytes: batch, token, head
  int64_t db, dt, dh;  // output strides
};

struct RopeParams {
  RopeTensor q, k;
  const int64_t* pos;
  int64_t pb, pt;  // position strides in elements
  const double* freq;
  int64_t rows, T;
  LaunchDiv by_half, by_tok, by_head;  // planes; a token's and a head's items
  int nq, nk, D, rot, tok;
  float amp, sign;
  bool stream;
};

template <int DT, int N> struct RopeVec {
  typename Elem<DT>::T e[N];
};

// N elements as one access: from an address that is a multiple of their size (WIDE), or of one
// element's.
template <int DT, int N, bool WIDE>
__device__ __forceinline__ RopeVec<DT, N> rope_load(const char* p) {
  RopeVec<DT, N> v;
  constexpr int B = N * (int)sizeof(v.e[0]), A = WIDE ? (B < 16 ? B : 16) : (int)sizeof(v.e[0]);
  __builtin_memcpy(&v, __builtin_assume_aligned(p, A), B);
  return v;
}
template <int DT, int N, bool WIDE>
__device__ __forceinline__ void rope_store(char* p, const RopeVec<DT, N>& v, bool stream) {
  constexpr int B = N * (int)sizeof(v.e[0]), A = WIDE ? (B < 16 ? B : 16) : (int)sizeof(v.e[0]);
  if constexpr (WIDE && B == 16) {
    if (stream) {
      __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), (u32x4*)p);
      return;
    }
  }
  __builtin_memcpy(__builtin_assume_aligned(p, A), &v, B);
}

template <int DT, int VP, bool IL>
__global__ void __launch_bounds__(RP_NT) rope_kernel(RopeParams p) {
  constexpr int ES = (int)sizeof(typename Elem<DT>::T);
  __shared__ __attribute__((aligned(16))) float s_cos[RP_MAX_TRIG], s_sin[RP_MAX_TRIG];
  __shared__ int64_t s_at[RP_MAX_TOK][4];  // a token's offsets into q, k and the outputs
  const int half = p.rot / 2;
  const int64_t row0 = (int64_t)blockIdx.x * p.tok;
  const int ntok = (int)min((int64_t)p.tok, p.rows - row0);
  if (threadIdx.x < ntok) {
    const int64_t row = row0 + threadIdx.x, b = row / p.T, t = row - b * p.T;
    int64_t* at = s_at[threadIdx.x];
    at[0] = b * p.q.sb + t * p.q.st;
    at[1] = b * p.q.db + t * p.q.dt;
    at[2] = b * p.k.sb + t * p.k.st;
    at[3] = b * p.k.db + t * p.k.dt;
  }
  for (int i = threadIdx.x; i < ntok * half; i += RP_NT) {
    const int t = (int)p.by_half.div(i), j = i - t * half;
    const int64_t row = row0 + t, b = row / p.T;
    const double pos = (double)p.pos[b * p.pb + (row - b * p.T) * p.pt];
    const double turns = pos * (p.freq[j] * 0.15915494309189533577);  // 1 / (2 pi)
    const float r = (float)(turns - rint(turns));
    float s, c;
    sincospif(2.0f * r, &s, &c);
    s_cos[i] = c * p.amp;
    s_sin[i] = s * p.amp * p.sign;
  }
  __syncthreads();

  // Items of a token: heads x (half / VP vectors or pairs of vectors to turn, then the tail's
  // vectors, as wide as those).
  constexpr bool WIDE = VP > 1;
  constexpr int TV = IL && WIDE ? 2 * VP : VP;
  const int nrot = half / VP;
  const int n_items = ntok * (int)p.by_tok.d;
  // RP_BATCH items' loads are issued before the first one's store (a store to what may be the
  // same memory holds later loads back): 32 KiB in flight a CU do not cover HBM's latency.
  using First = RopeVec<DT, IL ? 2 * VP : VP>;
  for (int i0 = threadIdx.x; i0 < n_items; i0 += RP_BATCH * RP_NT) {
    First va[RP_BATCH];
    RopeVec<DT, VP> vb[RP_BATCH];  // the other half's planes
    char* dst[RP_BATCH];
    int trig[RP_BATCH];  // where the item's planes begin in the tables, -1: a tail vector
#pragma unroll
    for (int k = 0; k < RP_BATCH; ++k) {
      const int i = min(i0 + k * RP_NT, n_items - 1);
      const int t = (int)p.by_tok.div(i), u = i - t * (int)p.by_tok.d;
      int h = (int)p.by_head.div(u);
      const int c = u - h * (int)p.by_head.d;
      const bool is_k = h >= p.nq;
      if (is_k) h -= p.nq;
      const char* src =
          is_k ? p.k.src + s_at[t][2] + h * p.k.sh : p.q.src + s_at[t][0] + h * p.q.sh;
      dst[k] = is_k ? p.k.dst + s_at[t][3] + h * p.k.dh : p.q.dst + s_at[t][1] + h * p.q.dh;
      trig[k] = c < nrot ? t * half + c * VP : -1;
      const int64_t off = (int64_t)(c < nrot ? c * (IL ? 2 * VP : VP) : p.rot + (c - nrot) * TV) * ES;
      dst[k] += off;
      if (VP == 1 && IL && c >= nrot) va[k].e[0] = rope_load<DT, 1, WIDE>(src + off).e[0];
      else va[k] = rope_load<DT, IL ? 2 * VP : VP, WIDE>(src + off);
      if (!IL && c < nrot) vb[k] = rope_load<DT, VP, WIDE>(src + off + (int64_t)half * ES);
    }
#pragma unroll
    for (int k = 0; k < RP_BATCH; ++k) {
      if (i0 + k * RP_NT >= n_items) break;
      if (trig[k] < 0) {
        RopeVec<DT, TV> v;
#pragma unroll
        for (int e = 0; e < TV; ++e) v.e[e] = va[k].e[e];
        rope_store<DT, TV, WIDE>(dst[k], v, p.stream);
        continue;
      }
      const float *cs = s_cos + trig[k], *sn = s_sin + trig[k];
      float oa[VP], ob[VP];
#pragma unroll
      for (int e = 0; e < VP; ++e) {
        const float x1 = Elem<DT>::to_f(va[k].e[IL ? 2 * e : e]);
        const float x2 = Elem<DT>::to_f(IL ? va[k].e[IL ? 2 * e + 1 : e] : vb[k].e[e]);
        oa[e] = x1 * cs[e] - x2 * sn[e];
        ob[e] = x2 * cs[e] + x1 * sn[e];
      }
      if constexpr (IL) {
        float o[2 * VP];
#pragma unroll
        for (int e = 0; e < VP; ++e) o[2 * e] = oa[e], o[2 * e + 1] = ob[e];
        round_to<DT>(o, va[k].e);
        rope_store<DT, 2 * VP, WIDE>(dst[k], va[k], p.stream);
      } else {
        round_to<DT>(oa, va[k].e);
        round_to<DT>(ob, vb[k].e);
        rope_store<DT, VP, WIDE>(dst[k], va[k], p.stream);
        rope_store<DT, VP, WIDE>(dst[k] + (int64_t)half * ES, vb[k], p.stream);
      }
    }
  }
}

// vp: planes of a thread and step, 16 bytes' worth (8 or 4 elements; half as many pairs) or a
// half of that, or one.
template <int DT, bool IL>
static void rope_run(const RopeParams& P, int vp, unsigned grid, hipStream_t s) {
  constexpr int W = 16 / (int)sizeof(typename Elem<DT>::T) / (IL ? 2 : 1);
  if (vp == W) rope_kernel<DT, W, IL><<<grid, RP_NT, 0, s>>>(P);
  else if (W > 2 && vp == W / 2) rope_kernel<DT, (W > 2 ? W / 2 : 1), IL><<<grid, RP_NT, 0, s>>>(P);
  else rope_kernel<DT, 1, IL><<<grid, RP_NT, 0, s>>>(P);
}

template <int DT>
static int rope_launch(const RopeParams& P, int vp, bool il, unsigned grid, hipStream_t s) {
  KernelTimer timer("rope", s);
  if (il) rope_run<DT, true>(P, vp, grid, s);
  else rope_run<DT, false>(P, vp, grid, s);
  timer.stop();
  return check_launch("rope_kernel");
}

}  // namespace nsmoe

using namespace nsmoe;

extern "C" int nsmoe_rope(const nsmoe_rope_args* a, void* stream) {
  NSMOE_REQUIRE(a, "rope: NULL args");
  NSMOE_REQUIRE(a->dtype >= DT_BF16 && a->dtype <= DT_F32, "rope: unknown dtype %d", a->dtype);
  NSMOE_REQUIRE(a->head_dim >= 1 && a->head_dim <= 1024, "rope: head_dim %d (need 1 .. 1024)",
                a->head_dim);
  NSMOE_REQUIRE(a->rot_dim >= 2 && a->rot_dim % 2 == 0 && a->rot_dim <= a->head_dim,
                "rope: rot_dim %d must be even, 2 .. head_dim (%d)", a->rot_dim, a->head_dim);
  NSMOE_REQUIRE(a->n_q >= 0 && a->n_k >= 0 && a->n_q <= 4096 && a->n_k <= 4096 &&
                    a->n_q + a->n_k >= 1,
                "rope: n_q %d and n_k %d (need 0 .. 4096, one of them not 0)", a->n_q, a->n_k);
  NSMOE_REQUIRE(a->batch >= 0 && a->n_tokens >= 0 && a->batch < INT32_MAX &&
                    a->n_tokens < INT32_MAX,
                "rope: bad batch / n_tokens");
  if (a->batch == 0 || a->n_tokens == 0) return NSMOE_OK;
  NSMOE_REQUIRE(a->positions && a->freqs && (!a->n_q || (a->q && a->q_out)) &&
                    (!a->n_k || (a->k && a->k_out)),
                "rope: NULL pointer");
  const int es = a->dtype == DT_F32 ? 4 : 2;
  RopeParams P{};
  // The widest vectors that the planes, the tail and every address allow, up to 16 bytes: the
  // planes of a thread and step are 16 bytes of each half of a head, or 16 bytes of pairs.
  uint64_t bits = 0;  // of every address and stride, in bytes
  auto take = [&](RopeTensor& t, const void* src, void* dst, const int64_t* si, const int64_t* so) {
    t = RopeTensor{(const char*)src, (char*)dst, si[0] * es, si[1] * es, si[2] * es,
                   so[0] * es, so[1] * es, so[2] * es};
    bits |= (uint64_t)src | (uint64_t)dst;
    for (int i = 0; i < 3; ++i) bits |= (uint64_t)(si[i] * es) | (uint64_t)(so[i] * es);
  };
  if (a->n_q) take(P.q, a->q, a->q_out, a->q_stride, a->q_out_stride);
  if (a->n_k) take(P.k, a->k, a->k_out, a->k_stride, a->k_out_stride);
  NSMOE_REQUIRE((bits & (uint64_t)(es - 1)) == 0, "rope: misaligned pointer");
  const bool il = a->interleaved != 0;
  const bool in_place = (!a->n_q || a->q == a->q_out) && (!a->n_k || a->k == a->k_out);
  const int half = a->rot_dim / 2, tail = a->head_dim - a->rot_dim;
  auto fits = [&](int vp) {
    const int unit = il ? 2 * vp : vp;  // elements of a vector
    return half % vp == 0 && (in_place || tail % unit == 0) && (bits & (uint64_t)(unit * es - 1)) == 0;
  };
  const int widest = 16 / es / (il ? 2 : 1);
  const int vp = fits(widest) ? widest : widest > 2 && fits(widest / 2) ? widest / 2 : 1;
  const int per_head = half / vp + (in_place ? 0 : tail / (il && vp > 1 ? 2 * vp : vp));
  P.by_half = launch_div(half);
  P.by_head = launch_div(per_head);
  P.by_tok = launch_div((int64_t)per_head * (a->n_q + a->n_k));
  P.pos = a->positions;
  P.pb = a->pos_stride[0];
  P.pt = a->pos_stride[1];
  P.freq = a->freqs;
  P.rows = a->batch * a->n_tokens;
  P.T = a->n_tokens;
  P.nq = a->n_q;
  P.nk = a->n_k;
  P.D = a->head_dim;
  P.rot = a->rot_dim;
  P.amp = a->amplitude;
  P.sign = a->inverse ? -1.0f : 1.0f;
  // Tokens per workgroup: as many as leave eight workgroups a CU (what fits at once), at most
  // 16 and what the LDS table holds.
  int64_t tok = P.rows / (8 * device_cus());
  tok = tok < 1 ? 1 : tok > RP_MAX_TOK ? RP_MAX_TOK : tok;
  if (tok > RP_MAX_TRIG / half) tok = RP_MAX_TRIG / half;
  P.tok = (int)tok;
  // Outputs that the 256 MiB memory-side cache cannot hold beside the inputs are stored past
  // it: 150 us against 161 for an fp32 forward and backward of 335 MB each; at 100 MB a call
  // 20.1 against 17.9, so smaller ones are not.
  P.stream = 2 * P.rows * (a->n_q + a->n_k) * (int64_t)a->head_dim * es > (256ll << 20);
  const int64_t grid = cdiv(P.rows, tok);
  NSMOE_REQUIRE(grid < INT32_MAX, "rope: grid too large");
  hipStream_t s = (hipStream_t)stream;
  switch (a->dtype) {
    case DT_BF16: return rope_launch<DT_BF16>(P, vp, il, (unsigned)grid, s);
    case DT_F16: return rope_launch<DT_F16>(P, vp, il, (unsigned)grid, s);
    default: return rope_launch<DT_F32>(P, vp, il, (unsigned)grid, s);
  }
}
