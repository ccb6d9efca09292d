// Attention of a batch's new tokens over a prefix that all sequences share and over each
// sequence's own cache (16-bit types, head dims 64 and 128).
//
// Query i < n of sequence b stands at row len_b - n + i of its own cache, behind the prefix's
// P keys; it sees the prefix and its own rows up to itself, within `window` keys (itself
// counted) when one is given:
//   o = sum_j p_j v_j,  p = softmax_j(scale q . k_j)  over both
// (reference: the grouped-query attention of src/model/mha.py:245-287; its decode loop,
// nanospeaker.py:233-237, holds the whole context once per sequence).
//
// The prefix's keys and values are one copy in memory, so they are multiplied once for the
// whole batch: for a key/value head the queries of ALL sequences and of its group are the
// columns of one product, and the prefix is read once instead of batch times.  The own rows
// are read by their sequence's columns alone.  Both are split over the keys into parts; a part
// leaves its columns' running maximum, sum and unnormalised output in fp32, and
// prefix_join_kernel joins them.  A decode step's short context takes one launch instead
// (prefix_whole_kernel), each sequence's columns over the prefix and its own rows.
//
// Two forms of a part, by the number of columns:
//   few   up to 32 columns (a decode step's own rows, or the prefix of a small batch): each
//         of the 4 waves takes 32-key tiles of its own through its own LDS buffers, with no
//         barrier in the loop; the waves' results are joined through LDS at the end.  Bound by
//         HBM: the keys and values are read once (64 x 640 rows of 8 heads of 128: 34 us,
//         4.9 TB/s).
//   many  64, 128 or 192 columns (the prefix under a batch, a prompt behind the prefix): the 4
//         waves share 64-key tiles and own different columns.  Bound by the vector work of the
//         softmax and the matrix products, which hardly overlap (VALU 57 %, MFMA 31 % busy): 6144
//         columns x 8192 keys x 3 heads of 64 take 56 us, 690 TFLOP/s.
//
// Layouts are the prefill kernel's (attention.hip): S^T = K Q^T, so that the probabilities of
// a column are already the B operand of O^T = V^T P^T, with V read by ds_read_b64_tr_b16 from
// tiles that LDS-DMA copied with a chunk swizzle.  Scores, maxima, sums and outputs are fp32;
// the probabilities enter the P V product rounded to the type (up to half a step each, the size
// of the output's own rounding; the few form, whose matrix pipe idles, multiplies the bf16
// remainders too), their sum is of the unrounded ones.
#include <algorithm>

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
  float* part_o;   // [rows][slots][D]
  float2* part_ml; // [rows][slots]: log2-scaled maximum, sum
  float* score;    // [B, Hkv, n G, spad] log2-scaled scores of the own rows, or NULL
  uint16_t* out;   // [rows, D]
  float* lse;      // [rows] or NULL
  const float* w_in;
  float* w_out;    // [B, Hkv, S]
  int B, n, P, S, Hq, Hkv, G, window, spad;
  int np, ns;            // parts of the prefix and of each own cache: a row's slots
  int chunk_p, chunk_s;  // keys per part
  int rbp, rbs;          // column blocks of a prefix part and of an own part
  int items_p;           // workgroups of the prefix (before the own ones)
  LaunchDiv by_G, by_n, by_seq, by_chunk;  // group's heads, new tokens, a sequence's rows, keys
  float scale_log2;
};

__device__ __forceinline__ int pa_len(const PrefixAttnParams& p, int b) {
  const int n = p.lens[b];
  return n < 0 ? 0 : n > p.S ? p.S : n;
}

// How many parts a sequence's own rows make: as many as the length is nearest to, of one size,
// because a short remainder would pay a part's start and end for little.  The parts from there
// to ns are not computed, and prefix_join_kernel does not look at them.
__device__ __forceinline__ int pa_parts_of(const PrefixAttnParams& p, int len) {
  return max(1, (int)p.by_chunk.div((uint32_t)(len + p.chunk_s / 2)));
}

// The sequence with the r-th longest cache (the earlier one first among equals), for up to 64
// sequences: the longest parts then start first, and the launch does not end on one that
// started late (64 ragged sequences of 256 to 1024 rows, dim 128: 39 us against 42 unordered).
// Lane l holds sequence l's length; the r-th largest is found bit by bit.
__device__ __forceinline__ int pa_by_length(const PrefixAttnParams& p, int r) {
  const int lane = threadIdx.x & 63;
  const int len = lane < p.B ? pa_len(p, lane) : -1;
  int v = 0;  // the largest value that more than r lengths reach
  for (int bit = 1 << (31 - __clz(p.S | 1)); bit; bit >>= 1)
    if (__popcll(__ballot(len >= v + bit)) > r) v += bit;
  const int k = r - (int)__popcll(__ballot(len > v));  // which of the equal ones
  const uint64_t same = __ballot(len == v);
  const bool me = len == v && (int)__popcll(same & (((uint64_t)1 << lane) - 1)) == k;
  return (int)__ffsll((unsigned long long)__ballot(me)) - 1;
}

// One part: a key/value head's columns against a run of keys.
struct PartJob {
  const uint16_t *k, *v;  // the head's row 0
  int64_t kt, vt;         // row strides
  int hk, b;              // b < 0: the prefix
  int col0, cols;         // first column, and how many columns there are in all
  int key0, key1;         // the part's keys
  int slot;               // -1: a part that this sequence does not have
};

__device__ __forceinline__ PartJob pa_job(const PrefixAttnParams& p, int item, bool own,
                                          int width) {
  PartJob j;
  if (!own) {
    // Column blocks of one run of keys follow each other and sit on one XCD: they read the
    // same keys and values from its L2.
    item = xcd_remap(item, p.items_p);
    const int rb = item % p.rbp;
    item /= p.rbp;
    const int split = item % p.np;
    j.hk = item / p.np;
    j.b = -1;
    j.k = p.kp + j.hk * p.kph;
    j.v = p.vp + j.hk * p.vph;
    j.kt = p.kpt;
    j.vt = p.vpt;
    j.col0 = rb * width;
    j.cols = p.B * p.n * p.G;
    j.key0 = split * p.chunk_p;
    j.key1 = j.key0 + p.chunk_p;
    j.slot = split;
  } else {
    // Parts in the order of their keys: the ones that short sequences leave empty come last.
    j.hk = item % p.Hkv;
    item /= p.Hkv;
    const int rb = item % p.rbs;
    item /= p.rbs;
    j.b = item % p.B;
    const int split = item / p.B;
    if (p.B > 1 && p.B <= 64) j.b = pa_by_length(p, j.b);
    j.k = p.k + j.b * p.kb + j.hk * p.kh;
    j.v = p.v + j.b * p.vb + j.hk * p.vh;
    j.kt = p.kt;
    j.vt = p.vt;
    j.col0 = rb * width;
    j.cols = p.n * p.G;
    const int len = pa_len(p, j.b), parts = pa_parts_of(p, len);
    // ceil(tiles / parts): exact, the quotient of two integers below 2^23 rounded once
    const int size = (int)((float)((len + 127) / 128 + parts - 1) / (float)parts) * 128;
    j.key0 = split * size;
    j.key1 = j.key0 + size;
    j.slot = split < parts ? p.np + split : -1;
  }
  return j;
}

// A column of a part: which row of q / out it is, and the keys [first, last] it sees, in the
// part's own numbering (none: last < first).
struct Column {
  int row;    // (b n + i) Hq + head, or -1 past the last column
  int64_t q;  // element offset into q
  int first, last;
};

// The keys that the query standing at row `at` of its cache sees, of the prefix or its own.
__device__ __forceinline__ void pa_sight(const PrefixAttnParams& p, bool own, int at, int& first,
                                         int& last) {
  const int me = own ? at : p.P + at;
  first = p.window ? max(0, me - p.window + 1) : 0;
  last = own ? at : p.P - 1;
  if (at < 0 || first > last) first = 0, last = -1;  // a query that has no row sees nothing
}

__device__ __forceinline__ Column pa_column(const PrefixAttnParams& p, const PartJob& j, int c) {
  Column r{-1, 0, 0, -1};
  if (c >= j.cols) return r;
  int i = (int)p.by_G.div(c), b = j.b;
  const int head = j.hk * p.G + c - i * p.G;
  if (b < 0) {
    b = (int)p.by_n.div(i);
    i -= b * p.n;
  }
  r.row = (b * p.n + i) * p.Hq + head;
  r.q = b * p.qb + i * p.qn + head * p.qh;
  pa_sight(p, j.b >= 0, pa_len(p, b) - p.n + i, r.first, r.last);
  return r;
}

// The keys [lo, hi) that some column of [col0, col0 + width) sees, within the part's.  Known
// without the columns where nothing but the part decides it, so that the first tiles can be on
// their way before the columns are looked at.
__device__ __forceinline__ void pa_range(const PrefixAttnParams& p, const PartJob& j, int width,
                                         int lane, int& lo, int& hi) {
  if (j.b >= 0) {  // one sequence: its columns are in the order of their queries
    const int at0 = pa_len(p, j.b) - p.n;
    int first, last;
    pa_sight(p, true, at0 + (int)p.by_G.div(min(j.col0 + width, j.cols) - 1), first, last);
    hi = last + 1;
    pa_sight(p, true, max(0, at0 + (int)p.by_G.div(j.col0)), lo, last);
  } else if (!p.window) {
    lo = 0;
    hi = p.P;
  } else {
    lo = INT32_MAX;
    hi = 0;
    for (int c = j.col0 + lane; c < min(j.col0 + width, j.cols); c += 64) {
      const Column k = pa_column(p, j, c);
      if (k.last < k.first) continue;
      lo = min(lo, k.first);
      hi = max(hi, k.last + 1);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      lo = min(lo, __shfl_xor(lo, o));
      hi = max(hi, __shfl_xor(hi, o));
    }
  }
  lo = __builtin_amdgcn_readfirstlane(max(lo, j.key0));
  hi = __builtin_amdgcn_readfirstlane(min(hi, j.key1));
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
// + 3 of column l16 of each block in o, and its own keys' part of the sum in l.  The exponents
// are taken against m, which moves only for a score that lies past `limit` (2^8 times m's
// exponential; any score while there is no m): the ratio of the sums is the same whatever m
// is, and p <= 256 stays well inside the types.  neg = -m log2(e) scale, 0 while there is no m.
template <int D, int NB>
struct PaState {
  f32x4 o[D / 16][NB];
  float m[NB], l[NB], limit[NB], neg[NB];
};

// A column's row, -1 for a padding column, PA_BLIND - row for one that sees nothing here.
constexpr int PA_BLIND = -2;

// The columns of a wave: query fragments, rows and key ranges.  SCORES: a form that calls with
// accumulated weights use (up to 64 columns), which leaves the scores of own rows behind.
template <int DT, int D, int NB, bool SCORES>
struct PaCols {
  typename Mma<DT>::Frag q[NB][D / 32];
  int row[NB], first[NB], last[NB];
  int all_first, all_last;          // keys within them every column sees
  float* score[SCORES ? NB : 1];  // this lane's column's scores (from key 0 on), or NULL
};

// The keys that every column of a wave sees.
template <int DT, int D, int NB, bool SC>
__device__ __forceinline__ void pa_common(PaCols<DT, D, NB, SC>& w) {
  int lo = w.first[0], hi = w.last[0];
#pragma unroll
  for (int nb = 1; nb < NB; ++nb) lo = max(lo, w.first[nb]), hi = min(hi, w.last[nb]);
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) lo = max(lo, __shfl_xor(lo, o)), hi = min(hi, __shfl_xor(hi, o));
  w.all_first = __builtin_amdgcn_readfirstlane(lo);
  w.all_last = __builtin_amdgcn_readfirstlane(hi);
}

template <int DT, int D, int NB, bool SC>
__device__ __forceinline__ void pa_load_cols(const PrefixAttnParams& p, const PartJob& j, int c0,
                                             int lane, PaCols<DT, D, NB, SC>& w) {
  const int l16 = lane & 15, g = lane >> 4;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int col = c0 + 16 * nb + l16;
    const Column c = pa_column(p, j, col);
    const bool live = c.last >= c.first;
    // A column that sees nothing, and a padding one, asks for no mask: its zero queries are
    // multiplied like any other's and what comes of it is dropped at the end.
    w.row[nb] = live || c.row < 0 ? c.row : PA_BLIND - c.row;
    w.first[nb] = c.first;
    w.last[nb] = live ? c.last : INT32_MAX;
#pragma unroll
    for (int ks = 0; ks < D / 32; ++ks) {
      u32x4 v = {0u, 0u, 0u, 0u};
      if (live) v = *(const u32x4*)(p.q + c.q + 32 * ks + 8 * g);
      w.q[nb][ks].v = v;
    }
    if constexpr (SC)
      w.score[nb] = p.score && j.b >= 0 && c.row >= 0
                        ? p.score + (((int64_t)j.b * p.Hkv + j.hk) * j.cols + col) * p.spad
                        : nullptr;
  }
  pa_common(w);
}

// A tile of KB * 16 keys from key0 on, in three steps.  Scores: S^T = K Q^T from the K rows in
// LDS; lane (g, l16) gets keys 16 kb + 4 g + e of column l16.
template <int DT, int D, int NB, int KB, bool SC>
__device__ __forceinline__ void pa_scores(const PaCols<DT, D, NB, SC>& w, const char* Kt, int lane,
                                          f32x4 (&s)[KB][NB]) {
  using M = Mma<DT>;
  constexpr int RB = 2 * D;  // bytes per row
  const int l16 = lane & 15, g = lane >> 4;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) s[kb][nb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int ks = 0; ks < D / 32; ++ks)
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int r = 16 * kb + l16;
      const typename M::Frag kf = M::load(Kt + r * RB + (((4 * ks + g) ^ pa_swz<D>(r)) << 4));
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) M::run(s[kb][nb], kf, w.q[nb][ks]);
    }
}

// Keys outside a column's range, or past `top`: one select per score, on tiles that cross some
// edge only.
template <int DT, int D, int NB, int KB, bool SC>
__device__ __forceinline__ void pa_mask(const PaCols<DT, D, NB, SC>& w, f32x4 (&s)[KB][NB], int key0,
                                        int lane, int top = INT32_MAX) {
  if (key0 >= w.all_first && key0 + 16 * KB - 1 <= min(w.all_last, top)) return;  // uniform
  const int g = lane >> 4;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = key0 + 16 * kb + 4 * g + e;
        const bool dead = (key < w.first[nb]) | (key > min(w.last[nb], top));
        s[kb][nb][e] = dead ? PA_NONE : s[kb][nb][e];
      }
}

// Leaves a tile's scores where they are asked for.
template <int DT, int D, int NB, int KB, bool SC>
__device__ __forceinline__ void pa_keep(const PaCols<DT, D, NB, SC>& w, const f32x4 (&s)[KB][NB],
                                        int key0, float c, int lane) {
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
    if (w.score[nb])
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
        *(f32x4*)(w.score[nb] + key0 + 16 * kb + 4 * (lane >> 4)) = s[kb][nb] * c;
}

// Turns masked scores into probabilities against the running reference, and sums them.
template <int D, int NB, int KB>
__device__ __forceinline__ void pa_softmax(PaState<D, NB>& st, f32x4 (&s)[KB][NB], float c) {
  float mx[NB];  // of this lane's keys
  bool past = false;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    mx[nb] = s[0][nb][0];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int e = 0; e < 4; ++e) mx[nb] = fmaxf(mx[nb], s[kb][nb][e]);
    past |= mx[nb] > st.limit[nb];
  }
  if (__ballot(past)) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const float top = pa_max4(mx[nb]);
      if (!(top > st.limit[nb])) continue;
      const float alpha =
          st.m[nb] == PA_NONE ? 0.0f : __builtin_amdgcn_exp2f((st.m[nb] - top) * c);
#pragma unroll
      for (int db = 0; db < D / 16; ++db) st.o[db][nb] *= alpha;
      st.l[nb] *= alpha;
      st.m[nb] = top;
      st.limit[nb] = top + 8.0f / c;
      st.neg[nb] = -(top * c);
    }
  }
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    float sum = 0.0f;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float pe = __builtin_amdgcn_exp2f(fmaf(s[kb][nb][e], c, st.neg[nb]));
        s[kb][nb][e] = pe;
        sum += pe;
      }
    st.l[nb] += sum;
  }
}

// O^T += V^T P^T, 32 keys at a time: slot 8 g + e is key 4 g + e, slot 8 g + 4 + e key
// 16 + 4 g + e, of P and of V alike.  With SPLIT the part of each probability that its rounding
// to the type leaves behind is multiplied too, rounded in its turn: up to 2^-16 of it is lost
// instead of 2^-8 (bf16).  In the many form that would cost a quarter (69 -> 85 us).
template <int DT, int D, int NB, int KB, bool SPLIT>
__device__ __forceinline__ void pa_values(PaState<D, NB>& st, const f32x4 (&s)[KB][NB],
                                          const char* Vt, int lane) {
  using M = Mma<DT>;
  using Frag = typename M::Frag;
  constexpr int RB = 2 * D;
  const int l16 = lane & 15, g = lane >> 4;
#pragma unroll
  for (int ks = 0; ks < KB / 2; ++ks) {
    Frag pf[NB], pr[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const f32x4 a = s[2 * ks][nb], b = s[2 * ks + 1][nb];
      pf[nb].v = u32x4{pack2<DT>(a[0], a[1]), pack2<DT>(a[2], a[3]), pack2<DT>(b[0], b[1]),
                       pack2<DT>(b[2], b[3])};
      if constexpr (SPLIT) {
        auto rest = [&](float x, float y, uint32_t hi) {
          return pack2<DT>(x - unpack2<DT>(hi, 0), y - unpack2<DT>(hi, 1));
        };
        pr[nb].v = u32x4{rest(a[0], a[1], pf[nb].v[0]), rest(a[2], a[3], pf[nb].v[1]),
                         rest(b[0], b[1], pf[nb].v[2]), rest(b[2], b[3], pf[nb].v[3])};
      }
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
      for (int nb = 0; nb < NB; ++nb) {
        M::run(st.o[db][nb], vf, pf[nb]);
        if constexpr (SPLIT) M::run(st.o[db][nb], vf, pr[nb]);
      }
    }
  }
}

template <int D, int NB>
__device__ __forceinline__ void pa_clear(PaState<D, NB>& st) {
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    st.m[nb] = st.limit[nb] = PA_NONE;
    st.l[nb] = st.neg[nb] = 0.0f;
#pragma unroll
    for (int db = 0; db < D / 16; ++db) st.o[db][nb] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
}

// LDS-DMA copies of a wave for one of K / V: N copies of 1 KiB (1024 / 2 D rows each) from row
// `row0` of a tile on, into LDS at `dst` plus 1 KiB each.  Rows outside [lo, hi) become zeros:
// what lies there was never written, and 0 * NaN is NaN.
template <int D, int N>
struct PaCopy {
  const uint16_t* src[N];  // this lane's chunk in tile 0
  int row[N];
  int64_t stride;

  __device__ __forceinline__ void set(const uint16_t* base, int64_t st, int row0, int lane) {
    constexpr int CPR = D / 8, RPC = 64 / CPR;  // chunks per row, rows per copy
    stride = st;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      row[u] = row0 + u * RPC + lane / CPR;
      src[u] = base + row[u] * st + ((lane % CPR) ^ pa_swz<D>(row[u])) * 8;
    }
  }
  __device__ __forceinline__ void issue(int key0, int keys, int lo, int hi, uint32_t dst,
                                        int lane) const {
    const int64_t off = (int64_t)key0 * stride;
    const bool whole = key0 >= lo && key0 + keys <= hi;  // uniform
    if (whole) {
#pragma unroll
      for (int u = 0; u < N; ++u) async_copy16_to(src[u] + off, dst + u * 1024);
      return;
    }
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const uint16_t* s = src[u] + off;
      if (key0 + row[u] < lo || key0 + row[u] >= hi)
        s = (const uint16_t*)((const char*)g_zero_kib + lane * 16);
      async_copy16_to(s, dst + u * 1024);
    }
  }
};

__device__ __forceinline__ uint32_t pa_lds(const char* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}

template <int D> struct PaGeo {
  static constexpr int FEW_KEYS = 32;
  static constexpr int FEW_TILE = FEW_KEYS * 2 * D;  // bytes of K or V
  static constexpr int FEW_LDS = 4 * 2 * FEW_TILE;   // 32 or 64 KiB
  static constexpr int MANY_KEYS = 64;
  static constexpr int MANY_STAGES = D == 64 ? 3 : 2;
  static constexpr int MANY_TILE = MANY_KEYS * 2 * D;
  static constexpr int MANY_LDS = MANY_STAGES * 2 * MANY_TILE;  // 48 or 64 KiB
};

// Joins NW waves through their buffers, 16 columns at a time, and calls
// emit(row, dim, maximum, sum, four dims of the output) for each column: the maximum is -inf for
// one that saw nothing.
template <int DT, int D, int NB, int NW, bool SC, class F>
__device__ __forceinline__ void pa_join_waves(const PrefixAttnParams& p,
                                              const PaCols<DT, D, NB, SC>& w,
                                              const PaState<D, NB>& st, char* lds, F&& emit) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, g = lane >> 4;
  float* s_o = (float*)lds;                      // [NW][16][D]
  float* s_m = (float*)(lds + NW * 16 * D * 4);  // [NW][16]
  float* s_l = s_m + NW * 16;                    // [NW][16]
  int* s_row = (int*)(s_l + NW * 16);            // [16]
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    float l = st.l[nb];
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    __syncthreads();
    if (g == 0) {
      s_m[wave * 16 + l16] = st.m[nb];
      s_l[wave * 16 + l16] = l;
      s_row[l16] = w.row[nb];
    }
#pragma unroll
    for (int db = 0; db < D / 16; ++db)
      *(f32x4*)(s_o + (wave * 16 + l16) * D + 16 * db + 4 * g) = st.o[db][nb];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * (D / 4); i += NW * 64) {
      const int col = i / (D / 4), d = (i % (D / 4)) * 4;
      const int r = s_row[col], row = r <= PA_BLIND ? PA_BLIND - r : r;
      if (row < 0) continue;
      float m = PA_NONE;
      if (r >= 0) {
#pragma unroll
        for (int k = 0; k < NW; ++k) m = fmaxf(m, s_m[k * 16 + col]);
      }
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
      float sum = 0.0f;
      if (m != PA_NONE) {
#pragma unroll
        for (int k = 0; k < NW; ++k) {
          const float mk = s_m[k * 16 + col];
          if (mk == PA_NONE) continue;
          const float f = __builtin_amdgcn_exp2f((mk - m) * p.scale_log2);
          sum += s_l[k * 16 + col] * f;
          o += *(const f32x4*)(s_o + (k * 16 + col) * D + d) * f;
        }
      }
      emit(row, d, m, sum, o);
    }
  }
}

template <int DT, int D, int NB>
__device__ void pa_few(const PrefixAttnParams& p, const PartJob& j, char* lds) {
  using Geo = PaGeo<D>;
  constexpr int KEYS = Geo::FEW_KEYS, TILE = Geo::FEW_TILE, KB = KEYS / 16;
  constexpr int NC = TILE / 1024;  // copies of one of K / V per tile
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int lo, hi;
  pa_range(p, j, 16 * NB, lane, lo, hi);
  // One buffer each for K and V, a wave's own: the next tile's K is copied from when this
  // one's scores are done, its V from when this one's product is.  What hides the copies'
  // latency is the other waves of the CU (8 to 16, each with 8 or 16 KiB of tile).
  char* Kt = lds + wave * 2 * TILE;
  char* Vt = Kt + TILE;
  const uint32_t kd = pa_lds(Kt), vd = kd + TILE;
  PaCopy<D, NC> ck, cv;
  ck.set(j.k, j.kt, 0, lane);
  cv.set(j.v, j.vt, 0, lane);
  int t = lo / KEYS + wave;
  const int t1 = hi > lo ? (hi + KEYS - 1) / KEYS : 0;
  if (t < t1) {
    ck.issue(t * KEYS, KEYS, lo, hi, kd, lane);
    cv.issue(t * KEYS, KEYS, lo, hi, vd, lane);
  }
  PaCols<DT, D, NB, true> w;
  pa_load_cols(p, j, j.col0, lane, w);
  wait_vmcnt<0>();  // see pa_many
  PaState<D, NB> st;
  pa_clear(st);
  // Scores that are asked for are stored a tile late, after a wait that has given the copies
  // time: stores count with the copies, and the waits below would stand still for fresh ones.
  const bool keep = p.score && j.b >= 0;
  f32x4 raw[KB][NB];
  int raw_at = -1;
  for (; t < t1; t += 4) {
    f32x4 s[KB][NB];
    wait_vmcnt<NC>();  // this tile's K; its V stays in flight
    asm volatile("" ::: "memory");
    if (keep && raw_at >= 0) pa_keep(w, raw, raw_at, p.scale_log2, lane);
    pa_scores(w, Kt, lane, s);
    asm volatile("" ::: "memory");
    wait_lgkm0();      // K has been read
    const bool more = t + 4 < t1;
    if (more) ck.issue((t + 4) * KEYS, KEYS, lo, hi, kd, lane);
    pa_mask(w, s, t * KEYS, lane);
    if (keep) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) raw[kb][nb] = s[kb][nb];
      raw_at = t * KEYS;
    }
    pa_softmax(st, s, p.scale_log2);
    if (more) wait_vmcnt<NC>();  // this tile's V; the next K stays in flight
    else wait_vmcnt<0>();
    asm volatile("" ::: "memory");
    pa_values<DT, D, NB, KB, DT == DT_BF16>(st, s, Vt, lane);
    asm volatile("" ::: "memory");
    wait_lgkm0();      // V has been read
    if (more) cv.issue((t + 4) * KEYS, KEYS, lo, hi, vd, lane);
  }

  if (keep && raw_at >= 0) pa_keep(w, raw, raw_at, p.scale_log2, lane);

  const int64_t slots = p.np + p.ns;
  pa_join_waves<DT, D, NB, 4>(p, w, st, lds, [&](int row, int d, float m, float sum,
                                                const f32x4& o) {
    const int64_t at = row * slots + j.slot;
    if (m != PA_NONE) *(f32x4*)(p.part_o + at * D + d) = o;
    if (d == 0) p.part_ml[at] = make_float2(m * p.scale_log2, sum);
  });
}

template <int DT, int D, int NB>
__device__ void pa_many(const PrefixAttnParams& p, const PartJob& j, char* lds) {
  using Geo = PaGeo<D>;
  constexpr int KEYS = Geo::MANY_KEYS, ST = Geo::MANY_STAGES, TILE = Geo::MANY_TILE;
  constexpr int KB = KEYS / 16;
  constexpr int NC = TILE / 1024 / 4;  // copies of one of K / V per tile and wave
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int lo, hi;
  pa_range(p, j, 64 * NB, lane, lo, hi);
  const uint32_t lds0 = pa_lds(lds) + (uint32_t)(wave * NC * 1024);
  PaCopy<D, NC> ck, cv;
  constexpr int ROWS = KEYS / 4;  // rows that a wave copies
  ck.set(j.k, j.kt, wave * ROWS, lane);
  cv.set(j.v, j.vt, wave * ROWS, lane);
  auto issue = [&](int t, int stage) {
    const uint32_t dst = lds0 + (uint32_t)(stage * 2 * TILE);
    ck.issue(t * KEYS, KEYS, lo, hi, dst, lane);
    cv.issue(t * KEYS, KEYS, lo, hi, dst + TILE, lane);
  };
  const int t0 = hi > lo ? lo / KEYS : 0, t1 = hi > lo ? (hi + KEYS - 1) / KEYS : 0;
#pragma unroll
  for (int u = 0; u < ST - 1; ++u)
    if (t0 + u < t1) issue(t0 + u, u);
  PaCols<DT, D, NB, NB == 1> w;
  pa_load_cols(p, j, j.col0 + wave * 16 * NB, lane, w);
  // The queries are waited for here: left to their first use, the compiler would put its wait,
  // which knows nothing of the copies, into the loop and drain them at every tile.
  wait_vmcnt<0>();
  PaState<D, NB> st;
  pa_clear(st);
  int stage = 0;
  for (int t = t0; t < t1; ++t) {
    // this wave's copies of tile t; with three stages tile t + 1's stay in flight
    if (ST == 3 && t + 1 < t1) wait_vmcnt<2 * NC>();
    else wait_vmcnt<0>();
    asm volatile("" ::: "memory");
    wait_lgkm0();   // this wave's LDS reads of the stage that is copied into next
    barrier_dma();  // every wave's copies of tile t; every wave done with tile t - 1
    if (t + ST - 1 < t1) issue(t + ST - 1, (stage + ST - 1) % ST);
    const char* tile = lds + stage * 2 * TILE;
    f32x4 s[KB][NB];
    pa_scores(w, tile, lane, s);
    pa_mask(w, s, t * KEYS, lane);
    if constexpr (NB == 1) pa_keep(w, s, t * KEYS, p.scale_log2, lane);
    pa_softmax(st, s, p.scale_log2);
    pa_values<DT, D, NB, KB, false>(st, s, tile + TILE, lane);
    stage = stage + 1 == ST ? 0 : stage + 1;
  }
  wait_vmcnt<0>();
  const int slots = p.np + p.ns;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    float l = st.l[nb];
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    const int r = w.row[nb], row = r <= PA_BLIND ? PA_BLIND - r : r;
    if (row < 0) continue;
    const int64_t at = (int64_t)row * slots + j.slot;
    const float m = r >= 0 ? st.m[nb] : PA_NONE;
    if (g == 0) p.part_ml[at] = make_float2(m * p.scale_log2, l);
    if (m == PA_NONE) continue;
    float* dst = p.part_o + at * D + 4 * g;
#pragma unroll
    for (int db = 0; db < D / 16; ++db) *(f32x4*)(dst + 16 * db) = st.o[db][nb];
  }
}

// A short context in one launch, without parts: a workgroup takes the columns, up to 16 NB, of
// one sequence and key/value head over the prefix and then its own rows, its eight waves the
// 32-key tiles of both in turn as in pa_few, and writes the output.  Keys are numbered through:
// own row r is key P + r, and a column sees one run of them.  Bound by latency: a launch, the
// lengths, the queries and a round of tiles after the other.  Eight waves take half the rounds of
// four (512 + 1024 keys, dim 64: 9.6 us against 11.8) and fill 64 or 128 KiB of LDS.
constexpr int PA_WHOLE_WAVES = 8;

template <int DT, int D, int NB>
__global__ void __launch_bounds__(PA_WHOLE_WAVES * 64, 2) prefix_whole_kernel(PrefixAttnParams p) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  using Geo = PaGeo<D>;
  constexpr int KEYS = Geo::FEW_KEYS, TILE = Geo::FEW_TILE, KB = KEYS / 16;
  constexpr int NC = TILE / 1024, NW = PA_WHOLE_WAVES;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  PartJob j{};
  j.hk = (int)blockIdx.x % p.Hkv;
  j.b = (int)blockIdx.x / p.Hkv;
  j.cols = p.n * p.G;
  j.key1 = p.S;
  int lo, hi;  // own rows that some column sees
  pa_range(p, j, 16 * NB, lane, lo, hi);
  const int at0 = max(0, pa_len(p, j.b) - p.n);  // the first query's row
  const int lo_p = p.window ? min(p.P, max(0, p.P + at0 - p.window + 1)) : 0;
  const int tp0 = lo_p / KEYS, ts0 = lo / KEYS;
  const int tp = hi > lo ? (p.P + KEYS - 1) / KEYS - tp0 : 0;
  const int tiles = hi > lo ? tp + (hi + KEYS - 1) / KEYS - ts0 : 0;
  const uint16_t *kp = p.kp + j.hk * p.kph, *vp = p.vp + j.hk * p.vph;
  const uint16_t *ko = p.k + j.b * p.kb + j.hk * p.kh, *vo = p.v + j.b * p.vb + j.hk * p.vh;
  char* Kt = lds + wave * 2 * TILE;
  char* Vt = Kt + TILE;
  const uint32_t kd = pa_lds(Kt), vd = kd + TILE;
  auto copy = [&](int i, const uint16_t* prefix, int64_t prefix_rows, const uint16_t* cache,
                  int64_t cache_rows, uint32_t dst) {
    PaCopy<D, NC> c;
    const bool own = i >= tp;
    c.set(own ? cache : prefix, own ? cache_rows : prefix_rows, 0, lane);
    const int tile = own ? ts0 + i - tp : tp0 + i;
    c.issue(tile * KEYS, KEYS, own ? lo : lo_p, own ? hi : p.P, dst, lane);
  };
  auto copy_k = [&](int i) { copy(i, kp, p.kpt, ko, p.kt, kd); };
  auto copy_v = [&](int i) { copy(i, vp, p.vpt, vo, p.vt, vd); };
  int t = wave;
  if (t < tiles) {
    copy_k(t);
    copy_v(t);
  }
  PaCols<DT, D, NB, false> w;
  pa_load_cols(p, j, 0, lane, w);
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
    if (w.row[nb] >= 0) {  // its own rows so far
      w.first[nb] = p.window ? p.P + w.last[nb] - p.window + 1 : 0;
      w.last[nb] += p.P;
    }
  pa_common(w);
  wait_vmcnt<0>();  // see pa_many
  PaState<D, NB> st;
  pa_clear(st);
  for (; t < tiles; t += NW) {
    f32x4 s[KB][NB];
    wait_vmcnt<NC>();  // this tile's K; its V stays in flight
    asm volatile("" ::: "memory");
    pa_scores(w, Kt, lane, s);
    asm volatile("" ::: "memory");
    wait_lgkm0();      // K has been read
    const bool more = t + NW < tiles;
    if (more) copy_k(t + NW);
    if (t < tp) pa_mask(w, s, (tp0 + t) * KEYS, lane, p.P - 1);
    else pa_mask(w, s, p.P + (ts0 + t - tp) * KEYS, lane);
    pa_softmax(st, s, p.scale_log2);
    if (more) wait_vmcnt<NC>();  // this tile's V; the next K stays in flight
    else wait_vmcnt<0>();
    asm volatile("" ::: "memory");
    pa_values<DT, D, NB, KB, DT == DT_BF16>(st, s, Vt, lane);
    asm volatile("" ::: "memory");
    wait_lgkm0();      // V has been read
    if (more) copy_v(t + NW);
  }
  pa_join_waves<DT, D, NB, NW>(p, w, st, lds, [&](int row, int d, float m, float sum, f32x4 o) {
    if (m != PA_NONE) o *= 1.0f / sum;
    *(uint2*)(p.out + (int64_t)row * D + d) =
        make_uint2(pack2<DT>(o[0], o[1]), pack2<DT>(o[2], o[3]));
    if (p.lse && d == 0)
      p.lse[row] = m == PA_NONE ? PA_NONE
                                : (m * p.scale_log2 + log2f(sum)) * 0.69314718055994531f;
  });
}

// Forms: 0, 1 few with 1 or 2 column blocks; 2, 3, 4 many with 1, 2 or 3 per wave.
constexpr int PA_FORMS = 5;
constexpr int PA_WIDTH[PA_FORMS] = {16, 32, 64, 128, 192};

template <int DT, int D, int FORM>
__device__ __forceinline__ void pa_part(const PrefixAttnParams& p, int item, bool own, char* lds) {
  const PartJob j = pa_job(p, item, own, PA_WIDTH[FORM]);
  if (j.slot < 0) return;
  if constexpr (FORM < 2) pa_few<DT, D, FORM + 1>(p, j, lds);
  else pa_many<DT, D, FORM - 1>(p, j, lds);
}

// The parts of the prefix (form FP) and, behind them, those of the own caches (form FS) in one
// launch: the first are bound by arithmetic under a batch, the second by HBM.  FP or FS -1:
// none of that kind.
template <int DT, int D, int FP, int FS>
__global__ void __launch_bounds__(PA_NT, 2) prefix_part_kernel(PrefixAttnParams p) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int item = (int)blockIdx.x;
  if constexpr (FP >= 0) {
    if (FS < 0 || item < p.items_p) {
      pa_part<DT, D, FP>(p, item, false, lds);
      return;
    }
  }
  if constexpr (FS >= 0) pa_part<DT, D, FS>(p, item - (FP >= 0 ? p.items_p : 0), true, lds);
}

// A wave's view of a row's parts: the log2-scaled maximum and the sum over all of them (-inf
// and 0 for a row that saw nothing), and this lane's factors 2^(m_s - m) for slots lane and
// 64 + lane (0 for a part that saw nothing).
struct PaTotal {
  float m, l, f0, f1;
};
constexpr int PA_MAX_SLOTS = 128;

__device__ __forceinline__ PaTotal pa_total(const PrefixAttnParams& p, int64_t row, int lane) {
  const int slots = p.np + p.ns;
  const float2* ml = p.part_ml + row * slots;
  const float2 none = make_float2(PA_NONE, 0.0f);
  float2 a = lane < slots ? ml[lane] : none, b = lane + 64 < slots ? ml[lane + 64] : none;
  // Slots of parts that the sequence does not have were not written: read (beside the length)
  // and dropped.
  if (p.ns > 1) {
    const int live = p.np + pa_parts_of(p, pa_len(p, (int)p.by_seq.div((uint32_t)row)));
    if (lane >= live) a = none;
    if (lane + 64 >= live) b = none;
  }
  PaTotal r;
  r.m = fmaxf(a.x, b.x);
  for (int o = 32; o; o >>= 1) r.m = fmaxf(r.m, __shfl_xor(r.m, o));
  r.f0 = a.x == PA_NONE ? 0.0f : __builtin_amdgcn_exp2f(a.x - r.m);
  r.f1 = b.x == PA_NONE ? 0.0f : __builtin_amdgcn_exp2f(b.x - r.m);
  r.l = a.y * r.f0 + b.y * r.f1;
  for (int o = 32; o; o >>= 1) r.l += __shfl_xor(r.l, o);
  return r;
}

// Joins the parts: a wave per row of the output, D / 4 lanes on a part, 64 / (D / 4) parts at
// once.  The workgroups behind those of the rows add each cached key's weight:
// w_out = w_in + sum over its columns of 2^(score - log2 total).
constexpr int PA_JOIN_KEYS = 4 * PA_NT;

template <int DT, int D>
__global__ void __launch_bounds__(PA_NT) prefix_join_kernel(PrefixAttnParams p, int row_blocks) {
  constexpr int LPR = D / 4, NG = 64 / LPR;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if ((int)blockIdx.x < row_blocks) {
    const int64_t row = (int64_t)blockIdx.x * 4 + wave;
    if (row >= (int64_t)p.B * p.n * p.Hq) return;
    const int slots = p.np + p.ns, grp = lane / LPR, d = (lane % LPR) * 4;
    const PaTotal t = pa_total(p, row, lane);
    const float* po = p.part_o + row * slots * D + d;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    // Four loads in flight a lane.  A part that saw nothing has factor 0 and was not written.
    for (int s0 = 0; s0 < slots; s0 += 4 * NG) {
      float f[4];
      f32x4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int s = s0 + u * NG;
        f[u] = __shfl(s < 64 ? t.f0 : t.f1, (s & 63) + grp);
        if (s >= PA_MAX_SLOTS) f[u] = 0.0f;
        v[u] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (f[u] != 0.0f) v[u] = *(const f32x4*)(po + (int64_t)(s + grp) * D);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) o += v[u] * f[u];
    }
#pragma unroll
    for (int x = LPR; x < 64; x <<= 1)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], x);
    if (grp) return;
    if (t.m != PA_NONE) o *= 1.0f / t.l;
    *(uint2*)(p.out + row * D + d) = make_uint2(pack2<DT>(o[0], o[1]), pack2<DT>(o[2], o[3]));
    if (p.lse && d == 0)
      p.lse[row] = t.m == PA_NONE ? PA_NONE : (t.m + log2f(t.l)) * 0.69314718055994531f;
    return;
  }
  // A workgroup takes PA_JOIN_KEYS keys of one (sequence, key/value head).
  __shared__ float s_total[64];
  const int chunks = (p.S + PA_JOIN_KEYS - 1) / PA_JOIN_KEYS;
  int it = (int)blockIdx.x - row_blocks;
  const int chunk = it % chunks;
  it /= chunks;
  const int hk = it % p.Hkv, b = it / p.Hkv;
  const int cols = p.n * p.G;
  for (int c = wave; c < cols; c += 4) {
    const PaTotal t =
        pa_total(p, ((int64_t)b * p.n + c / p.G) * p.Hq + hk * p.G + c % p.G, lane);
    if (lane == 0) s_total[c] = t.m == PA_NONE ? INFINITY : t.m + log2f(t.l);  // 2^(x - inf) = 0
  }
  __syncthreads();
  const int row0 = pa_len(p, b) - p.n, key0 = chunk * PA_JOIN_KEYS + threadIdx.x;
  const int64_t head = (int64_t)b * p.Hkv + hk;
  constexpr int KPT = PA_JOIN_KEYS / PA_NT;
  float sum[KPT], before[KPT];  // the new weights are added up before they meet the old
#pragma unroll
  for (int u = 0; u < KPT; ++u) {
    const int key = key0 + u * PA_NT;
    before[u] = p.w_in && key < p.S ? p.w_in[head * p.S + key] : 0.0f;
    sum[u] = 0.0f;
  }
  // Only the columns that see a key: their scores alone were written.
  for (int c = 0; c < cols; ++c) {
    const int at = row0 + (int)p.by_G.div(c);
    const float* sc = p.score + (head * cols + c) * p.spad;
    const float total = s_total[c];
    float x[KPT];
#pragma unroll
    for (int u = 0; u < KPT; ++u) {
      const int key = key0 + u * PA_NT;
      x[u] = key <= at && (!p.window || at - key < p.window) ? sc[key] : PA_NONE;
    }
#pragma unroll
    for (int u = 0; u < KPT; ++u) sum[u] += __builtin_amdgcn_exp2f(x[u] - total);
  }
#pragma unroll
  for (int u = 0; u < KPT; ++u) {
    const int key = key0 + u * PA_NT;
    if (key < p.S) p.w_out[head * p.S + key] = before[u] + sum[u];
  }
}

// ---- host -------------------------------------------------------------------------------

struct PrefixPlan {
  bool whole;          // no parts: prefix_whole_kernel
  int form_p, form_s;  // -1: no such parts
  int np, ns, chunk_p, chunk_s, rbp, rbs, spad;
  int64_t items_p, items_s, rows;
  size_t off_ml, off_score, bytes;
};

// The narrowest form that takes the columns in one block; past 128 the widest one (192 columns
// at head dim 64, 128 at 128, whose accumulators take the registers).
static int pa_form(int64_t cols, int D) {
  for (int f = 0; f < 4; ++f)
    if (cols <= PA_WIDTH[f]) return f;
  return D == 64 ? 4 : 3;
}

static PrefixPlan pa_plan(const nsmoe_prefix_attn_args* a) {
  PrefixPlan pl{};
  const int64_t G = a->n_heads / a->n_kv_heads, B = a->batch, n = a->n_new, D = a->head_dim;
  const int64_t cus = device_cus(), slots = 2 * cus;  // workgroups that run at once
  pl.rows = B * n * a->n_heads;
  // A short context is not split: up to 1536 keys of 64 dims or 768 of 128 that a sequence sees,
  // while every workgroup has its CU (or half of one, at 64) at once.  4 sequences of 512 + 64
  // keys, dim 64: 7.2 us in a graph and 11.3 called eagerly against 8.7 and 15.2 in parts, 64 of
  // 512 + 1024 12.4 and 12.3 against 14.6 and 16.1; a single one of 2048 + 256 12.8 against 9.1.
  const int64_t all = a->prefix_len + a->cap;
  const int64_t seen = a->window ? std::min<int64_t>(all, a->window + n - 1) : all;
  if (a->cap > 0 && n * G <= 32 && !a->weights_out && seen * D <= 1536 * 64 &&
      B * a->n_kv_heads * D <= slots * 64) {
    pl.whole = true;
    return pl;
  }
  pl.form_p = a->prefix_len > 0 ? pa_form(B * n * G, a->head_dim) : -1;
  pl.form_s = a->cap > 0 ? pa_form(n * G, a->head_dim) : -1;
  // What the two kinds of parts take, roughly, in us on the whole chip: the bytes of their keys
  // and values at 5 TB/s (the caches half full) or their products at 600 TFLOP/s.
  auto cost = [&](double keys, double cols) {
    return std::max(keys * a->n_kv_heads * D * 4 / 5e6, keys * cols * a->n_kv_heads * D * 4 / 6e8);
  };
  const double cost_p = cost((double)a->prefix_len, (double)(B * n * G));
  const double cost_s = cost(0.5 * (double)(a->cap * B), (double)(n * G));
  // Keys per part: whole turns of four 32-key tiles, at most 64 parts.
  auto chunk_of = [&](int64_t keys, int64_t parts) {
    parts = parts < 1 ? 1 : parts > 64 ? 64 : parts;
    return (int)(cdiv(cdiv(keys, parts), 128) * 128);
  };
  if (pl.form_p >= 0) {
    // The prefix's parts take their share of the chip beside the caches' (64 sequences behind
    // 8192 rows, dim 128, 1024-row caches: 128 to 192 of 512 workgroups 53 us, 512 of them 70).
    // Under many columns a part pays for its columns' loads and its output with 512 keys of
    // work, or 256 while there are fewer parts than CUs (that prefix alone: 24 us at 512 keys
    // a part, 33 at 1024, 27 at 256).
    pl.rbp = (int)cdiv(B * n * G, PA_WIDTH[pl.form_p]);
    const int64_t groups = (int64_t)pl.rbp * a->n_kv_heads, keys = a->prefix_len;
    int64_t parts = (int64_t)((double)slots * cost_p / (cost_p + cost_s) / groups + 0.5);
    if (pl.form_p < 2) parts *= 2;
    else parts = std::min(parts, std::max(keys / 512, std::min(keys / 256, cus / groups)));
    pl.chunk_p = chunk_of(keys, parts);
    pl.np = (int)cdiv(keys, pl.chunk_p);
    pl.items_p = pl.np * groups;
  }
  if (pl.form_s >= 0) {
    // About 768 keys a part, or fewer while that leaves slots empty: a part's start and end cost
    // about 2 us of its slot, and larger ones leave ragged lengths uneven (48 sequences of up to
    // 8191 rows, dim 64, with weights: 52 us; 55 at 1024 keys, 57 at 1280.  32 x 2048 rows, dim
    // 128: 44 us; 46 at 1024 and at 512).
    pl.rbs = (int)cdiv(n * G, PA_WIDTH[pl.form_s]);
    const int64_t groups = B * pl.rbs * a->n_kv_heads;
    pl.chunk_s = chunk_of(a->cap, std::max(cdiv(a->cap, 768), slots / groups));
    pl.ns = (int)cdiv(a->cap, pl.chunk_s);
    pl.items_s = pl.ns * groups;
  }
  pl.spad = (int)(cdiv(a->cap, 64) * 64);
  const size_t parts = (size_t)(pl.np + pl.ns), rows = (size_t)pl.rows;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  pl.off_ml = up(parts * rows * a->head_dim * 4);
  pl.off_score = pl.off_ml + up(parts * rows * 8);
  pl.bytes = pl.off_score;
  if (a->weights_out) pl.bytes += up((size_t)B * a->n_kv_heads * n * G * pl.spad * 4);
  return pl;
}

template <int DT, int D, int FP, int FS>
static int pa_run(const PrefixAttnParams& P, int64_t items, hipStream_t s) {
  constexpr int few = PaGeo<D>::FEW_LDS, many = PaGeo<D>::MANY_LDS;
  constexpr int lds = (FP >= 2 || FS >= 2) && many > few ? many
                      : (FP >= 0 && FP < 2) || (FS >= 0 && FS < 2) ? few : many;
  static_assert(PA_WIDTH[2] == 64, "weights stay within the forms that keep scores");
  static_assert(2 * 64 <= PA_MAX_SLOTS, "a lane holds two slots");
  static_assert(4 * 16 * (D * 4 + 8) + 64 <= few, "the join of the waves fits their buffers");
  NSMOE_REQUIRE(items < INT32_MAX, "prefix_attention: grid too large");
  KernelTimer timer("prefix_part", s);
  prefix_part_kernel<DT, D, FP, FS><<<(unsigned)items, PA_NT, lds, s>>>(P);
  timer.stop();
  return check_launch("prefix_part_kernel");
}

// Calls f with the form as a constant.
template <int D, class F>
static int pa_with_form(int form, F&& f) {
  switch (form) {
    case 0: return f(std::integral_constant<int, 0>{});
    case 1: return f(std::integral_constant<int, 1>{});
    case 2: return f(std::integral_constant<int, 2>{});
    case 3: return f(std::integral_constant<int, 3>{});
    default:
      if constexpr (D == 64) return f(std::integral_constant<int, 4>{});
      else return f(std::integral_constant<int, 3>{});
  }
}

template <int DT, int D>
static int pa_launch(const PrefixAttnParams& P, const PrefixPlan& pl, hipStream_t s) {
  if (pl.whole) {
    const unsigned grid = (unsigned)(P.B * P.Hkv);
    constexpr int NW = PA_WHOLE_WAVES, lds = NW * 2 * PaGeo<D>::FEW_TILE;
    static_assert(NW * 16 * (D * 4 + 8) + 64 <= lds, "the join of the waves fits their buffers");
    KernelTimer timer("prefix_whole", s);
    if (P.n * P.G <= 16) prefix_whole_kernel<DT, D, 1><<<grid, NW * 64, lds, s>>>(P);
    else prefix_whole_kernel<DT, D, 2><<<grid, NW * 64, lds, s>>>(P);
    timer.stop();
    return check_launch("prefix_whole_kernel");
  }
  // One launch for both kinds (a cache's columns are some of the prefix's: FS <= FP).
  const int64_t items = pl.items_p + pl.items_s;
  if (pl.form_p >= 0 && pl.form_s >= 0) {
    NSMOE_TRY(pa_with_form<D>(pl.form_p, [&](auto fp) {
      return pa_with_form<D>(pl.form_s, [&](auto fs) {
        constexpr int FP = decltype(fp)::value, FS = decltype(fs)::value;
        if constexpr (FS <= FP) return pa_run<DT, D, FP, FS>(P, items, s);
        else return (int)NSMOE_EINVAL;
      });
    }));
  } else if (pl.form_p >= 0) {
    NSMOE_TRY(pa_with_form<D>(pl.form_p, [&](auto fp) {
      return pa_run<DT, D, decltype(fp)::value, -1>(P, items, s);
    }));
  } else if (pl.form_s >= 0) {
    NSMOE_TRY(pa_with_form<D>(pl.form_s, [&](auto fs) {
      return pa_run<DT, D, -1, decltype(fs)::value>(P, items, s);
    }));
  }
  const int64_t row_blocks = cdiv(pl.rows, 4);
  int64_t grid = row_blocks;
  if (P.w_out) grid += (int64_t)P.B * P.Hkv * cdiv(P.S, PA_JOIN_KEYS);
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
  P.chunk_p = pl.chunk_p;
  P.chunk_s = pl.chunk_s;
  P.rbp = pl.rbp;
  P.rbs = pl.rbs;
  P.items_p = (int)pl.items_p;
  P.by_G = launch_div(P.G);
  P.by_n = launch_div(P.n);
  P.by_seq = launch_div((int64_t)P.n * P.Hq);
  P.by_chunk = launch_div(P.chunk_s > 0 ? P.chunk_s : 1);
  P.scale_log2 = a->scale * 1.4426950408889634f;
  hipStream_t s = (hipStream_t)stream;
  if (a->head_dim == 64)
    return a->dtype == DT_BF16 ? pa_launch<DT_BF16, 64>(P, pl, s) : pa_launch<DT_F16, 64>(P, pl, s);
  return a->dtype == DT_BF16 ? pa_launch<DT_BF16, 128>(P, pl, s) : pa_launch<DT_F16, 128>(P, pl, s);
}
