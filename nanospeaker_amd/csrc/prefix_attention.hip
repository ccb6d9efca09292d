// Attention of a batch's new tokens over a prefix that all sequences share and over each
// sequence's own cache (16-bit types, head dims 64 and 128).
//
// Query i < n of sequence b stands at row len_b - n + i of its own cache, behind the prefix's
// P keys; it sees the prefix and its own rows up to itself, within `window` keys (itself
// counted) when one is given:
//   o = sum_j p_j v_j,  p = softmax_j(scale q . k_j)  over both
// (reference: the grouped-query attention of src/model/mha.py:245-287 with a cache).
//
// The prefix's keys and values are one copy in memory, so they are multiplied once for the
// whole batch: for a key/value head the queries of ALL sequences and of its group are the
// columns of one product, and the prefix is read once instead of batch times.  The own rows
// are read by their sequence's columns alone.  Both are split over the keys into parts; a part
// leaves its columns' running maximum, sum and unnormalised output in fp32, and
// prefix_join_kernel joins them.
//
// Two forms of a part, by the number of columns:
//   few   up to 32 columns (a decode step's own rows, or the prefix of a small batch): each
//         of the 4 waves takes 32-key tiles of its own through its own LDS ring, with no
//         barrier in the loop; the waves' results are joined through LDS at the end.  Bound by
//         HBM: the keys and values are read once.
//   many  64 columns per column block of the waves (the prefix under a batch, a prompt behind
//         the prefix): the 4 waves share 64-key tiles and own different columns.  Bound by
//         the matrix products and the softmax between them.
//
// Layouts are the prefill kernel's (attention.hip): S^T = K Q^T, so that the probabilities of
// a column are already the B operand of O^T = V^T P^T, with V read by ds_read_b64_tr_b16 from
// tiles that LDS-DMA copied with a chunk swizzle.  Scores, maxima, sums and outputs are fp32;
// the probabilities enter the P V product rounded to the type (relative error up to half a
// step each, of the size of the output's own rounding), their sum is of the unrounded ones.
#include "../../include/nsmoe.h"
#include "gemm_core.h"
#include "nsmoe_capi_internal.h"

namespace nsmoe {

constexpr int PA_NT = 256;
constexpr float PA_NONE = -INFINITY;

struct PrefixAttnParams {
  const uint16_t *q, *kp, *vp, *k, *v;
  int64_t qb, qn, qh;          // q strides in elements: batch, token, head
  int64_t kpt, kph, vpt, vph;  // prefix: row, head
  int64_t kb, kt, kh, vb, vt, vh;
  const int32_t* lens;
  float* part_o;   // [slots][rows][D]
  float2* part_ml; // [slots][rows]: log2-scaled maximum, sum
  float* score;    // [B, Hkv, n G, spad] log2-scaled scores of the own rows, or NULL
  uint16_t* out;   // [rows, D]
  float* lse;      // [rows] or NULL
  const float* w_in;
  float* w_out;    // [B, Hkv, S]
  int B, n, P, S, Hq, Hkv, G, window, spad;
  int np, ns;      // parts of the prefix and of each own cache
  int rbp, rbs;    // column blocks of a prefix part and of an own part
  int items_p;     // workgroups of the prefix (before the own ones)
  float scale_log2;
};

__device__ __forceinline__ int pa_len(const PrefixAttnParams& p, int b) {
  const int n = p.lens[b];
  return n < 0 ? 0 : n > p.S ? p.S : n;
}

// One part: a key/value head's columns against a run of keys.
struct PartJob {
  const uint16_t *k, *v;  // the head's row 0
  int64_t kt, vt;         // row strides
  int hk, b;              // b < 0: the prefix
  int col0, cols;         // first column, and how many columns there are in all
  int split, splits, slot;
};

__device__ __forceinline__ PartJob pa_job(const PrefixAttnParams& p, int item, bool own,
                                          int width) {
  PartJob j;
  if (!own) {
    j.split = item % p.np;
    item /= p.np;
    const int rb = item % p.rbp;
    j.hk = item / p.rbp;
    j.b = -1;
    j.k = p.kp + j.hk * p.kph;
    j.v = p.vp + j.hk * p.vph;
    j.kt = p.kpt;
    j.vt = p.vpt;
    j.col0 = rb * width;
    j.cols = p.B * p.n * p.G;
    j.splits = p.np;
    j.slot = j.split;
  } else {
    j.split = item % p.ns;
    item /= p.ns;
    const int rb = item % p.rbs;
    item /= p.rbs;
    j.hk = item % p.Hkv;
    j.b = item / p.Hkv;
    j.k = p.k + j.b * p.kb + j.hk * p.kh;
    j.v = p.v + j.b * p.vb + j.hk * p.vh;
    j.kt = p.kt;
    j.vt = p.vt;
    j.col0 = rb * width;
    j.cols = p.n * p.G;
    j.splits = p.ns;
    j.slot = p.np + j.split;
  }
  return j;
}

// A column of a part: which row of q / out it is, and the keys [first, last] it sees, in the
// part's own numbering (none: last < first).
struct Column {
  int64_t row;  // (b n + i) Hq + head, or -1 past the last column
  int64_t q;    // element offset into q
  int first, last;
};

__device__ __forceinline__ Column pa_column(const PrefixAttnParams& p, const PartJob& j, int c) {
  Column r{-1, 0, 0, -1};
  if (c >= j.cols) return r;
  const int g = c % p.G;
  int i = c / p.G, b = j.b;
  if (b < 0) {
    b = i / p.n;
    i -= b * p.n;
  }
  const int head = j.hk * p.G + g;
  r.row = ((int64_t)b * p.n + i) * p.Hq + head;
  r.q = b * p.qb + i * p.qn + head * p.qh;
  const int at = pa_len(p, b) - p.n + i;  // the query's own row
  if (at < 0) return r;                   // a query that has no row sees nothing
  if (j.b < 0) {
    r.last = p.P - 1;
    r.first = p.window ? max(0, p.P + at - p.window + 1) : 0;
  } else {
    r.last = at;
    r.first = p.window ? max(0, at - p.window + 1) : 0;
  }
  if (r.first > r.last) r.first = 0, r.last = -1;
  return r;
}

// Chunk swizzle of a row of 2 D bytes (D / 8 chunks of 16): chunk c of row r sits at slot
// c ^ pa_swz(r), so that a fragment read (16 rows, one chunk) and a transposed read (8 rows x
// 32 bytes) fall on distinct banks.
template <int D>
__device__ __forceinline__ int pa_swz(int r) {
  if constexpr (D == 64) return (((r >> 1) & 3) << 1) | ((r >> 3) & 1);
  else return ((r & 7) << 1) | ((r >> 3) & 1);
}

__device__ __forceinline__ float pa_max4(float v) {  // over lanes l, l ^ 16, l ^ 32, l ^ 48
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// A wave's running state over NB blocks of 16 columns: lane (g, l16) holds dims 16 db + 4 g ..
// + 3 of column l16 of each block in o, and its own keys' part of the sum in l.
template <int D, int NB>
struct PaState {
  f32x4 o[D / 16][NB];
  float m[NB], l[NB];
};

// The columns of a wave: query fragments and key ranges.
template <int DT, int D, int NB>
struct PaCols {
  typename Mma<DT>::Frag q[NB][D / 32];
  int first[NB], last[NB];
};

template <int DT, int D, int NB>
__device__ __forceinline__ void pa_load_cols(const PrefixAttnParams& p, const PartJob& j, int c0,
                                             int lane, PaCols<DT, D, NB>& w, int& lo, int& hi) {
  const int l16 = lane & 15, g = lane >> 4;
  lo = INT32_MAX;
  hi = 0;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const Column c = pa_column(p, j, c0 + 16 * nb + l16);
    w.first[nb] = c.first;
    w.last[nb] = c.last;
    const bool live = c.last >= c.first;
    if (live) {
      lo = min(lo, c.first);
      hi = max(hi, c.last + 1);
    }
#pragma unroll
    for (int ks = 0; ks < D / 32; ++ks) {
      u32x4 v = {0u, 0u, 0u, 0u};
      if (live) v = *(const u32x4*)(p.q + c.q + 32 * ks + 8 * g);
      w.q[nb][ks].v = v;
    }
  }
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    lo = min(lo, __shfl_xor(lo, o));
    hi = max(hi, __shfl_xor(hi, o));
  }
  lo = min(lo, hi);  // nothing seen: an empty range
}

// One tile of KB * 16 keys from key0 on: scores, online softmax, P V.  Kt / Vt: the tile's rows
// in LDS.  `score`: where to leave this lane's column's scaled scores (its tile's key 0), or
// NULL per block.
template <int DT, int D, int NB, int KB>
__device__ __forceinline__ void pa_tile(const PaCols<DT, D, NB>& w, PaState<D, NB>& st,
                                        const char* Kt, const char* Vt, int key0, float c,
                                        int lane, float* const (&score)[NB]) {
  using M = Mma<DT>;
  using Frag = typename M::Frag;
  constexpr int RB = 2 * D;  // bytes per row
  const int l16 = lane & 15, g = lane >> 4;
  f32x4 s[KB][NB];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) s[kb][nb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int ks = 0; ks < D / 32; ++ks)
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int r = 16 * kb + l16;
      const Frag kf = M::load(Kt + r * RB + (((4 * ks + g) ^ pa_swz<D>(r)) << 4));
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) M::run(s[kb][nb], kf, w.q[nb][ks]);
    }
  // Keys outside a column's range: one select per score, on tiles that cross some edge only.
  bool edge = false;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) edge |= w.first[nb] > key0 || w.last[nb] < key0 + 16 * KB - 1;
  if (__ballot(edge)) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key0 + 16 * kb + 4 * g + e;
          const bool dead = (key < w.first[nb]) | (key > w.last[nb]);
          s[kb][nb][e] = dead ? PA_NONE : s[kb][nb][e];
        }
  }
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    if (score[nb]) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) *(f32x4*)(score[nb] + 16 * kb + 4 * g) = s[kb][nb] * c;
    }
    float mx = st.m[nb];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int e = 0; e < 4; ++e) mx = fmaxf(mx, s[kb][nb][e]);
    mx = pa_max4(mx);
    // The exponents' reference moves only past 2^8, or on the first finite score (the same
    // ratio whatever it is; p <= 256 stays well inside the types).
    const bool move = st.m[nb] == PA_NONE ? mx != PA_NONE : (mx - st.m[nb]) * c > 8.0f;
    if (__ballot(move)) {
      const float mnew = move ? mx : st.m[nb];
      const float alpha =
          st.m[nb] == PA_NONE ? 0.0f : __builtin_amdgcn_exp2f((st.m[nb] - mnew) * c);
#pragma unroll
      for (int db = 0; db < D / 16; ++db) st.o[db][nb] *= alpha;
      st.l[nb] *= alpha;
      st.m[nb] = mnew;
    }
    const float msub = st.m[nb] == PA_NONE ? 0.0f : st.m[nb] * c;
    float sum = 0.0f;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float pe = __builtin_amdgcn_exp2f(fmaf(s[kb][nb][e], c, -msub));
        s[kb][nb][e] = pe;
        sum += pe;
      }
    st.l[nb] += sum;
  }
  // O^T += V^T P^T, 32 keys at a time: slot 8 g + e is key 4 g + e, slot 8 g + 4 + e key
  // 16 + 4 g + e, of P and of V alike.
#pragma unroll
  for (int ks = 0; ks < KB / 2; ++ks) {
    Frag pf[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const f32x4 a = s[2 * ks][nb], b = s[2 * ks + 1][nb];
      pf[nb].v = u32x4{pack2<DT>(a[0], a[1]), pack2<DT>(a[2], a[3]), pack2<DT>(b[0], b[1]),
                       pack2<DT>(b[2], b[3])};
    }
    const int ra = 32 * ks + 4 * g + (l16 >> 2), rb = ra + 16;
    const int sub = (l16 & 3) >> 1, within = 8 * (l16 & 1);
#pragma unroll
    for (int db = 0; db < D / 16; ++db) {
      const int cc = 2 * db + sub;
      const uint2 lo = lds_read_tr16(Vt + ra * RB + ((cc ^ pa_swz<D>(ra)) << 4) + within);
      const uint2 hi = lds_read_tr16(Vt + rb * RB + ((cc ^ pa_swz<D>(rb)) << 4) + within);
      Frag vf;
      vf.v = u32x4{lo.x, lo.y, hi.x, hi.y};
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) M::run(st.o[db][nb], vf, pf[nb]);
    }
  }
}

template <int D, int NB>
__device__ __forceinline__ void pa_clear(PaState<D, NB>& st) {
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    st.m[nb] = PA_NONE;
    st.l[nb] = 0.0f;
#pragma unroll
    for (int db = 0; db < D / 16; ++db) st.o[db][nb] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
}

// LDS-DMA of `rows` rows from row key0 on of one of K / V into LDS at `dst`, rows outside
// [lo, hi) as zeros (what lies there was never written, and 0 * NaN is NaN).  A copy is 1 KiB.
template <int D>
__device__ __forceinline__ void pa_copy(const uint16_t* base, int64_t stride, int row, int key0,
                                        int lo, int hi, uint32_t dst, int lane) {
  constexpr int CPR = D / 8;  // chunks per row
  const int r = row + lane / CPR;
  const int c = (lane % CPR) ^ pa_swz<D>(r);
  const int key = key0 + r;
  const uint16_t* src = base + (int64_t)key * stride + c * 8;
  if (key < lo || key >= hi) src = (const uint16_t*)((const char*)g_zero_kib + lane * 16);
  async_copy16_to(src, dst);
}

__device__ __forceinline__ uint32_t pa_lds(const char* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}

template <int D> struct PaGeo {
  static constexpr int FEW_KEYS = 32;
  static constexpr int FEW_STAGES = D == 64 ? 3 : 2;
  static constexpr int FEW_TILE = FEW_KEYS * 2 * D;                    // bytes of K or V
  static constexpr int FEW_LDS = 4 * FEW_STAGES * 2 * FEW_TILE;
  static constexpr int MANY_KEYS = 64;
  static constexpr int MANY_STAGES = D == 64 ? 3 : 2;
  static constexpr int MANY_TILE = MANY_KEYS * 2 * D;
  static constexpr int MANY_LDS = MANY_STAGES * 2 * MANY_TILE;
};

// The split's run of key tiles: [lo, hi) cut into whole tiles from lo's tile on, dealt evenly.
__device__ __forceinline__ void pa_range(int lo, int hi, int tile, const PartJob& j, int& t0,
                                         int& t1) {
  const int a = lo / tile, b = hi > lo ? (hi + tile - 1) / tile : a;
  const int per = (b - a + j.splits - 1) / j.splits;
  t0 = min(b, a + j.split * per);
  t1 = min(b, t0 + per);
}

template <int DT, int D, int NB>
__device__ void pa_few(const PrefixAttnParams& p, const PartJob& j, char* lds) {
  using Geo = PaGeo<D>;
  constexpr int KEYS = Geo::FEW_KEYS, ST = Geo::FEW_STAGES, TILE = Geo::FEW_TILE;
  constexpr int RPC = 1024 / (2 * D);   // rows per copy
  constexpr int NC = KEYS / RPC;        // copies of one of K / V per tile
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  PaCols<DT, D, NB> w;
  int lo, hi, t0, t1;
  pa_load_cols<DT, D, NB>(p, j, j.col0, lane, w, lo, hi);
  lo = __builtin_amdgcn_readfirstlane(lo);
  hi = __builtin_amdgcn_readfirstlane(hi);
  pa_range(lo, hi, KEYS, j, t0, t1);
  float* score[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int col = j.col0 + 16 * nb + l16;
    score[nb] = p.score && j.b >= 0 && col < j.cols
                    ? p.score + (((int64_t)j.b * p.Hkv + j.hk) * j.cols + col) * p.spad
                    : nullptr;
  }
  // The columns' ranges may start late or end early: rows of a tile that no column sees are
  // not copied.  Padding columns see nothing and ask for no mask.
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
    if (j.col0 + 16 * nb + l16 >= j.cols) w.first[nb] = 0, w.last[nb] = INT32_MAX;

  char* ring = lds + wave * ST * 2 * TILE;
  const uint32_t ring0 = pa_lds(ring);
  auto issue = [&](int t, int stage) {
    const uint32_t dst = ring0 + (uint32_t)(stage * 2 * TILE);
#pragma unroll
    for (int u = 0; u < NC; ++u)
      pa_copy<D>(j.k, j.kt, u * RPC, t * KEYS, lo, hi, dst + u * 1024, lane);
#pragma unroll
    for (int u = 0; u < NC; ++u)
      pa_copy<D>(j.v, j.vt, u * RPC, t * KEYS, lo, hi, dst + TILE + u * 1024, lane);
  };
  PaState<D, NB> st;
  pa_clear(st);
  // Tiles wave, wave + 4, ...; ST - 1 of them in flight ahead of the one being multiplied.
#pragma unroll
  for (int u = 0; u < ST - 1; ++u)
    if (t0 + wave + 4 * u < t1) issue(t0 + wave + 4 * u, u);
  int stage = 0;
  for (int t = t0 + wave; t < t1; t += 4) {
    // The tile ST - 1 ahead goes into the stage that the previous turn has read: its LDS
    // reads have to be done (their results in registers) before the copy may land.
    asm volatile("" ::: "memory");
    wait_lgkm0();
    const int ahead = t + 4 * (ST - 1);
    if (ahead < t1) issue(ahead, (stage + ST - 1) % ST);
    // this tile's copies; those of the tiles behind it stay in flight
    const int later = min(ST - 1, (t1 - 1 - t) / 4);
    if (later == 0) wait_vmcnt<0>();
    else if (later == 1) wait_vmcnt<2 * NC>();
    else wait_vmcnt<4 * NC>();
    asm volatile("" ::: "memory");
    const char* tile = ring + stage * 2 * TILE;
    float* sc[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) sc[nb] = score[nb] ? score[nb] + t * KEYS : nullptr;
    pa_tile<DT, D, NB, KEYS / 16>(w, st, tile, tile + TILE, t * KEYS, p.scale_log2, lane, sc);
    stage = stage + 1 == ST ? 0 : stage + 1;
  }
  wait_vmcnt<0>();

  // Join the four waves: every wave's maximum, sum and output through LDS.
  __syncthreads();
  constexpr int W = 16 * NB;
  float* s_o = (float*)lds;                    // [4][W][D]
  float* s_m = (float*)(lds + 4 * W * D * 4);  // [4][W]
  float* s_l = s_m + 4 * W;                    // [4][W]
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    float l = st.l[nb];
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    const int col = 16 * nb + l16;
    if (g == 0) {
      s_m[wave * W + col] = st.m[nb];
      s_l[wave * W + col] = l;
    }
#pragma unroll
    for (int db = 0; db < D / 16; ++db)
      *(f32x4*)(s_o + (wave * W + col) * D + 16 * db + 4 * g) = st.o[db][nb];
  }
  __syncthreads();
  const int64_t rows = (int64_t)p.B * p.n * p.Hq;
  for (int i = threadIdx.x; i < W * (D / 4); i += PA_NT) {
    const int col = i / (D / 4), d = (i % (D / 4)) * 4;
    const Column c = pa_column(p, j, j.col0 + col);
    if (c.row < 0) continue;
    float m = PA_NONE;
#pragma unroll
    for (int k = 0; k < 4; ++k) m = fmaxf(m, s_m[k * W + col]);
    if (c.last < c.first) m = PA_NONE;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float l = 0.0f;
    if (m != PA_NONE) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float mk = s_m[k * W + col];
        if (mk == PA_NONE) continue;
        const float f = __builtin_amdgcn_exp2f((mk - m) * p.scale_log2);
        l += s_l[k * W + col] * f;
        o += *(const f32x4*)(s_o + (k * W + col) * D + d) * f;
      }
      *(f32x4*)(p.part_o + (j.slot * rows + c.row) * D + d) = o;
    }
    if (d == 0) p.part_ml[j.slot * rows + c.row] = make_float2(m * p.scale_log2, l);
  }
}

template <int DT, int D, int NB>
__device__ void pa_many(const PrefixAttnParams& p, const PartJob& j, char* lds) {
  using Geo = PaGeo<D>;
  constexpr int KEYS = Geo::MANY_KEYS, ST = Geo::MANY_STAGES, TILE = Geo::MANY_TILE;
  constexpr int RPC = 1024 / (2 * D);
  constexpr int NC = KEYS / RPC / 4;  // copies of one of K / V per tile and wave
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  __shared__ int s_lo[4], s_hi[4];
  PaCols<DT, D, NB> w;
  int lo, hi, t0, t1;
  const int c0 = j.col0 + wave * 16 * NB;
  pa_load_cols<DT, D, NB>(p, j, c0, lane, w, lo, hi);
  if (lane == 0) s_lo[wave] = hi > lo ? lo : INT32_MAX, s_hi[wave] = hi;
  __syncthreads();
  lo = min(min(s_lo[0], s_lo[1]), min(s_lo[2], s_lo[3]));
  hi = max(max(s_hi[0], s_hi[1]), max(s_hi[2], s_hi[3]));
  lo = __builtin_amdgcn_readfirstlane(min(lo, hi));
  hi = __builtin_amdgcn_readfirstlane(hi);
  pa_range(lo, hi, KEYS, j, t0, t1);
  float* score[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int col = c0 + 16 * nb + l16;
    score[nb] = p.score && j.b >= 0 && col < j.cols
                    ? p.score + (((int64_t)j.b * p.Hkv + j.hk) * j.cols + col) * p.spad
                    : nullptr;
    if (col >= j.cols) w.first[nb] = 0, w.last[nb] = INT32_MAX;
  }
  const uint32_t lds0 = pa_lds(lds);
  auto issue = [&](int t, int stage) {
    const uint32_t dst = lds0 + (uint32_t)(stage * 2 * TILE);
#pragma unroll
    for (int u = 0; u < NC; ++u) {
      const int cp = wave * NC + u;
      pa_copy<D>(j.k, j.kt, cp * RPC, t * KEYS, lo, hi, dst + cp * 1024, lane);
    }
#pragma unroll
    for (int u = 0; u < NC; ++u) {
      const int cp = wave * NC + u;
      pa_copy<D>(j.v, j.vt, cp * RPC, t * KEYS, lo, hi, dst + TILE + cp * 1024, lane);
    }
  };
  PaState<D, NB> st;
  pa_clear(st);
#pragma unroll
  for (int u = 0; u < ST - 1; ++u)
    if (t0 + u < t1) issue(t0 + u, u);
  int stage = 0;
  for (int t = t0; t < t1; ++t) {
    // this wave's copies of tile t; with three stages tile t + 1's stay in flight
    if (ST == 3 && t + 1 < t1) wait_vmcnt<2 * NC>();
    else wait_vmcnt<0>();
    asm volatile("" ::: "memory");
    wait_lgkm0();  // this wave's LDS reads of the stage that is copied into next
    barrier_dma();  // every wave's copies of tile t; every wave done with tile t - 1
    if (t + ST - 1 < t1) issue(t + ST - 1, (stage + ST - 1) % ST);
    const char* tile = lds + stage * 2 * TILE;
    float* sc[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) sc[nb] = score[nb] ? score[nb] + t * KEYS : nullptr;
    pa_tile<DT, D, NB, KEYS / 16>(w, st, tile, tile + TILE, t * KEYS, p.scale_log2, lane, sc);
    stage = stage + 1 == ST ? 0 : stage + 1;
  }
  wait_vmcnt<0>();
  const int64_t rows = (int64_t)p.B * p.n * p.Hq;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    float l = st.l[nb];
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    const Column c = pa_column(p, j, c0 + 16 * nb + l16);
    if (c.row < 0) continue;
    const float m = c.last < c.first ? PA_NONE : st.m[nb];
    if (g == 0) p.part_ml[j.slot * rows + c.row] = make_float2(m * p.scale_log2, l);
    if (m == PA_NONE) continue;
    float* dst = p.part_o + (j.slot * rows + c.row) * D + 4 * g;
#pragma unroll
    for (int db = 0; db < D / 16; ++db) *(f32x4*)(dst + 16 * db) = st.o[db][nb];
  }
}

// Forms: 0, 1 few with 1 or 2 column blocks; 2, 3 many with 1 or 2 per wave.
constexpr int PA_WIDTH[4] = {16, 32, 64, 128};

template <int DT, int D, int FORM>
__global__ void __launch_bounds__(PA_NT) prefix_part_kernel(PrefixAttnParams p, int own) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const PartJob j = pa_job(p, (int)blockIdx.x, own != 0, PA_WIDTH[FORM]);
  if constexpr (FORM < 2) pa_few<DT, D, FORM + 1>(p, j, lds);
  else pa_many<DT, D, FORM - 1>(p, j, lds);
}

// log2 of a row's whole sum of exponentials, from its parts; -inf for a row that saw nothing.
__device__ __forceinline__ void pa_total(const PrefixAttnParams& p, int64_t row, int64_t rows,
                                         float& m, float& l) {
  const int slots = p.np + p.ns;
  m = PA_NONE;
  for (int s = 0; s < slots; ++s) m = fmaxf(m, p.part_ml[s * rows + row].x);
  l = 0.0f;
  if (m == PA_NONE) return;
  for (int s = 0; s < slots; ++s) {
    const float2 ml = p.part_ml[s * rows + row];
    if (ml.x != PA_NONE) l += ml.y * __builtin_amdgcn_exp2f(ml.x - m);
  }
}

// Joins the parts: D / 4 lanes per row of the output.  The workgroups behind those of the rows
// add each cached key's weight: w_out = w_in + sum over its columns of 2^(score - log2 total).
template <int DT, int D>
__global__ void __launch_bounds__(PA_NT) prefix_join_kernel(PrefixAttnParams p, int row_blocks) {
  constexpr int LPR = D / 4, RPB = PA_NT / LPR;
  const int64_t rows = (int64_t)p.B * p.n * p.Hq;
  if ((int)blockIdx.x < row_blocks) {
    const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / LPR;
    if (row >= rows) return;
    const int d = (threadIdx.x % LPR) * 4;
    float m, l;
    pa_total(p, row, rows, m, l);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    if (m != PA_NONE)
      for (int s = 0; s < p.np + p.ns; ++s) {
        const float ms = p.part_ml[s * rows + row].x;
        if (ms == PA_NONE) continue;
        o += *(const f32x4*)(p.part_o + (s * rows + row) * D + d) *
             __builtin_amdgcn_exp2f(ms - m);
      }
    if (m != PA_NONE) o *= 1.0f / l;
    *(uint2*)(p.out + row * D + d) = make_uint2(pack2<DT>(o[0], o[1]), pack2<DT>(o[2], o[3]));
    if (p.lse && d == 0)
      p.lse[row] = m == PA_NONE ? PA_NONE : (m + log2f(l)) * 0.69314718055994531f;
    return;
  }
  // A workgroup takes PA_NT keys of one (sequence, key/value head).
  __shared__ float s_total[64];
  const int chunks = (p.S + PA_NT - 1) / PA_NT;
  int it = (int)blockIdx.x - row_blocks;
  const int chunk = it % chunks;
  it /= chunks;
  const int hk = it % p.Hkv, b = it / p.Hkv;
  const int cols = p.n * p.G;
  for (int c = threadIdx.x; c < cols; c += PA_NT) {
    float m, l;
    pa_total(p, ((int64_t)b * p.n + c / p.G) * p.Hq + hk * p.G + c % p.G, rows, m, l);
    s_total[c] = m == PA_NONE ? INFINITY : m + log2f(l);  // 2^(x - inf) = 0
  }
  __syncthreads();
  const int key = chunk * PA_NT + threadIdx.x;
  if (key >= p.S) return;
  const int64_t at = ((int64_t)b * p.Hkv + hk) * p.S + key;
  float w = p.w_in ? p.w_in[at] : 0.0f;
  // Only the columns that see the key: their scores alone were written.
  const float* sc = p.score + (((int64_t)b * p.Hkv + hk) * cols) * p.spad + key;
  const int row0 = pa_len(p, b) - p.n;
  float sum = 0.0f;
  for (int c = 0; c < cols; ++c) {
    const int at_q = row0 + c / p.G;
    if (at_q >= key && (!p.window || at_q - key < p.window))
      sum += __builtin_amdgcn_exp2f(sc[(int64_t)c * p.spad] - s_total[c]);
  }
  p.w_out[at] = w + sum;
}

// ---- host -------------------------------------------------------------------------------

struct PrefixPlan {
  int form_p, form_s;          // -1: no such parts
  int np, ns, rbp, rbs, spad;
  int64_t items_p, items_s, rows;
  size_t off_ml, off_score, bytes;
};

static int pa_form(int64_t cols) { return cols <= 16 ? 0 : cols <= 32 ? 1 : cols <= 64 ? 2 : 3; }

static PrefixPlan pa_plan(const nsmoe_prefix_attn_args* a) {
  PrefixPlan pl{};
  const int64_t G = a->n_heads / a->n_kv_heads, B = a->batch, n = a->n_new;
  const int64_t cus = device_cus();
  pl.rows = B * n * a->n_heads;
  pl.form_p = a->prefix_len > 0 ? pa_form(B * n * G) : -1;
  pl.form_s = a->cap > 0 ? pa_form(n * G) : -1;
  auto splits = [&](int64_t groups, int64_t keys) {
    // Two workgroups per CU over the launch; a part keeps at least two turns of the few
    // form's waves, or four tiles of the many form's.
    const int64_t least = 256;
    int64_t s = cdiv(2 * cus, groups), most = cdiv(keys, least);
    s = s < most ? s : most;
    return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
  };
  if (pl.form_p >= 0) {
    pl.rbp = (int)cdiv(B * n * G, PA_WIDTH[pl.form_p]);
    pl.np = splits((int64_t)pl.rbp * a->n_kv_heads, a->prefix_len);
    pl.items_p = (int64_t)pl.np * pl.rbp * a->n_kv_heads;
  }
  if (pl.form_s >= 0) {
    pl.rbs = (int)cdiv(n * G, PA_WIDTH[pl.form_s]);
    pl.ns = splits(B * pl.rbs * a->n_kv_heads, a->cap);
    pl.items_s = (int64_t)pl.ns * pl.rbs * a->n_kv_heads * B;
  }
  pl.spad = (int)(cdiv(a->cap, 64) * 64);
  const size_t slots = (size_t)(pl.np + pl.ns), rows = (size_t)pl.rows;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  pl.off_ml = up(slots * rows * a->head_dim * 4);
  pl.off_score = pl.off_ml + up(slots * rows * 8);
  pl.bytes = pl.off_score;
  if (a->weights_out) pl.bytes += up((size_t)B * a->n_kv_heads * n * G * pl.spad * 4);
  return pl;
}

template <int DT, int D, int FORM>
static int pa_part_form(const PrefixAttnParams& P, int64_t items, bool own, hipStream_t s) {
  constexpr int lds = FORM < 2 ? PaGeo<D>::FEW_LDS : PaGeo<D>::MANY_LDS;
  static_assert(FORM >= 2 || 4 * 16 * (FORM + 1) * (D * 4 + 8) <= lds, "the join fits the ring");
  prefix_part_kernel<DT, D, FORM><<<(unsigned)items, PA_NT, lds, s>>>(P, own);
  return check_launch("prefix_part_kernel");
}

template <int DT, int D>
static int pa_parts(const PrefixAttnParams& P, int form, int64_t items, bool own, hipStream_t s) {
  switch (form) {
    case 0: return pa_part_form<DT, D, 0>(P, items, own, s);
    case 1: return pa_part_form<DT, D, 1>(P, items, own, s);
    case 2: return pa_part_form<DT, D, 2>(P, items, own, s);
    default: return pa_part_form<DT, D, 3>(P, items, own, s);
  }
}

template <int DT, int D>
static int pa_launch(const PrefixAttnParams& P, const PrefixPlan& pl, hipStream_t s) {
  if (pl.form_p >= 0) {
    KernelTimer timer("prefix_part", s);
    NSMOE_TRY((pa_parts<DT, D>(P, pl.form_p, pl.items_p, false, s)));
    timer.stop();
  }
  if (pl.form_s >= 0) {
    KernelTimer timer("own_part", s);
    NSMOE_TRY((pa_parts<DT, D>(P, pl.form_s, pl.items_s, true, s)));
    timer.stop();
  }
  const int64_t row_blocks = cdiv(pl.rows, PA_NT / (D / 4));
  int64_t grid = row_blocks;
  if (P.w_out) grid += (int64_t)P.B * P.Hkv * cdiv(P.S, PA_NT);
  NSMOE_REQUIRE(grid < INT32_MAX, "prefix_attention: grid too large");
  KernelTimer timer("prefix_join", s);
  prefix_join_kernel<DT, D><<<(unsigned)grid, PA_NT, 0, s>>>(P, (int)row_blocks);
  timer.stop();
  return check_launch("prefix_join_kernel");
}

static int pa_check(const nsmoe_prefix_attn_args* a) {
  NSMOE_REQUIRE(a, "prefix_attention: NULL args");
  NSMOE_REQUIRE(a->dtype == DT_BF16 || a->dtype == DT_F16, "prefix_attention: 16-bit types only");
  NSMOE_REQUIRE(a->head_dim == 64 || a->head_dim == 128,
                "prefix_attention: head_dim must be 64 or 128 (got %d)", a->head_dim);
  NSMOE_REQUIRE(a->n_kv_heads >= 1 && a->n_heads >= a->n_kv_heads && a->n_heads <= 4096 &&
                    a->n_heads % a->n_kv_heads == 0,
                "prefix_attention: n_heads %d must be a multiple of n_kv_heads %d", a->n_heads,
                a->n_kv_heads);
  NSMOE_REQUIRE(a->batch >= 0 && a->n_new >= 0 && a->prefix_len >= 0 && a->cap >= 0 &&
                    a->prefix_len < (1 << 29) && a->cap < (1 << 29) && a->batch < (1 << 24) &&
                    a->n_new < (1 << 24) && a->batch * a->n_new * a->n_heads < (1 << 30),
                "prefix_attention: bad batch, new tokens, prefix or cache length");
  NSMOE_REQUIRE(a->window >= 0 && a->window < (1 << 30), "prefix_attention: window %d",
                a->window);
  NSMOE_REQUIRE(a->scale > 0.0f && a->scale < INFINITY, "prefix_attention: scale %g must be "
                "positive", (double)a->scale);
  NSMOE_REQUIRE(!a->weights_out || a->n_new * (a->n_heads / a->n_kv_heads) <= 64,
                "prefix_attention: weights for at most 64 query rows per key/value head (got "
                "%lld)", (long long)(a->n_new * (a->n_heads / a->n_kv_heads)));
  return NSMOE_OK;
}

}  // namespace nsmoe

using namespace nsmoe;

extern "C" size_t nsmoe_prefix_attention_workspace_size(const nsmoe_prefix_attn_args* a) {
  if (pa_check(a) != NSMOE_OK || a->batch == 0 || a->n_new == 0) return 0;
  return pa_plan(a).bytes;
}

extern "C" int nsmoe_prefix_attention(const nsmoe_prefix_attn_args* a, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  NSMOE_TRY(pa_check(a));
  if (a->batch == 0) return NSMOE_OK;
  NSMOE_REQUIRE(a->n_new >= 1, "prefix_attention: no new tokens");
  NSMOE_REQUIRE(a->q && a->out && a->lens && (a->prefix_len == 0 || (a->k_prefix && a->v_prefix)) &&
                    (a->cap == 0 || (a->k && a->v)),
                "prefix_attention: NULL pointer");
  uint64_t bits = (uint64_t)a->q | (uint64_t)a->out;
  for (int i = 0; i < 3; ++i) bits |= (uint64_t)(a->q_stride[i] * 2);
  if (a->prefix_len) {
    bits |= (uint64_t)a->k_prefix | (uint64_t)a->v_prefix;
    for (int i = 0; i < 2; ++i)
      bits |= (uint64_t)(a->kp_stride[i] * 2) | (uint64_t)(a->vp_stride[i] * 2);
  }
  if (a->cap) {
    bits |= (uint64_t)a->k | (uint64_t)a->v;
    for (int i = 0; i < 3; ++i)
      bits |= (uint64_t)(a->k_stride[i] * 2) | (uint64_t)(a->v_stride[i] * 2);
  }
  NSMOE_REQUIRE((bits & 15) == 0, "prefix_attention: pointers and strides must be multiples of 16 "
                                  "bytes");
  const PrefixPlan pl = pa_plan(a);
  NSMOE_REQUIRE(pl.items_p < INT32_MAX && pl.items_s < INT32_MAX,
                "prefix_attention: grid too large");
  if (workspace_bytes < pl.bytes || (pl.bytes && !workspace)) {
    set_error("prefix_attention: workspace of %zu bytes, need %zu", workspace_bytes, pl.bytes);
    return NSMOE_EWORKSPACE;
  }
  NSMOE_REQUIRE(((uintptr_t)workspace & 15) == 0, "prefix_attention: misaligned workspace");
  char* ws = (char*)workspace;
  PrefixAttnParams P{};
  P.q = (const uint16_t*)a->q;
  P.kp = (const uint16_t*)a->k_prefix;
  P.vp = (const uint16_t*)a->v_prefix;
  P.k = (const uint16_t*)a->k;
  P.v = (const uint16_t*)a->v;
  P.qb = a->q_stride[0], P.qn = a->q_stride[1], P.qh = a->q_stride[2];
  P.kpt = a->kp_stride[0], P.kph = a->kp_stride[1];
  P.vpt = a->vp_stride[0], P.vph = a->vp_stride[1];
  P.kb = a->k_stride[0], P.kt = a->k_stride[1], P.kh = a->k_stride[2];
  P.vb = a->v_stride[0], P.vt = a->v_stride[1], P.vh = a->v_stride[2];
  P.lens = a->lens;
  P.part_o = (float*)ws;
  P.part_ml = (float2*)(ws + pl.off_ml);
  P.score = a->weights_out ? (float*)(ws + pl.off_score) : nullptr;
  P.out = (uint16_t*)a->out;
  P.lse = a->lse;
  P.w_in = a->weights;
  P.w_out = a->weights_out;
  P.B = (int)a->batch;
  P.n = (int)a->n_new;
  P.P = (int)a->prefix_len;
  P.S = (int)a->cap;
  P.Hq = a->n_heads;
  P.Hkv = a->n_kv_heads;
  P.G = a->n_heads / a->n_kv_heads;
  P.window = a->window;
  P.spad = pl.spad;
  P.np = pl.np;
  P.ns = pl.ns;
  P.rbp = pl.rbp;
  P.rbs = pl.rbs;
  P.scale_log2 = a->scale * 1.4426950408889634f;
  hipStream_t s = (hipStream_t)stream;
  if (a->head_dim == 64)
    return a->dtype == DT_BF16 ? pa_launch<DT_BF16, 64>(P, pl, s) : pa_launch<DT_F16, 64>(P, pl, s);
  return a->dtype == DT_BF16 ? pa_launch<DT_BF16, 128>(P, pl, s) : pa_launch<DT_F16, 128>(P, pl, s);
}
