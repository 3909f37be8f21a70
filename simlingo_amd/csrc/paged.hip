// Operators over a paged key/value cache, for decoding many sequences that share a prompt (the questions and
// instructions about one camera frame, the beams of one answer). The greedy loop they stand beside re-runs one
// sequence (simlingo_training/models/language_model/llm.py:178-250); its cache is one sequence's rows (decode.hip).
//
//   slx_kv_append    rotates the new tokens' q and k (RoPE) and stores k and v in their pages, in one pass
//   slx_prefix_attn  attention of new tokens over a prefix that `width` sequences share and over each one's own keys
//
// A pool is a pair of bf16 arrays [page][slot][head][d] with any strides (d contiguous); a table row names the pages
// of one sequence in order. Table entries, positions and lengths are device data: what they get wrong (a page outside
// the pool, a position behind the table) is masked in the kernels and never read or written.
#include "common.h"
#include "../../include/slx.h"

namespace slx {

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

struct PoolView {
  bf16 *k, *v;
  long ps, ss, hs;  // element strides of a page, a slot, a head
  int n_pages, shift;
};

static int log2_exact(int x) {
  for (int s = 0; s < 31; ++s)
    if ((1 << s) == x) return s;
  return -1;
}

// ---- slx_kv_append ---------------------------------------------------------------------------------------------
// rotate_half RoPE: (x_j, x_{j + D/2}) -> (x_j cos - x_{j+D/2} sin, x_{j+D/2} cos + x_j sin), f32, rounded once.
// One thread takes the pair of 8-element chunks c and c + D/16 of one head (16-B loads and stores); a workgroup takes as many rows
// as fill it, so that neighbours read one row's cos and sin. Memory bound: 61 x 211 rows of 32 + 2 x 8 heads of 128, 317 MB in
// 60 us = 5.3 TB/s, the rate of a large copy. 798 rows of 14 + 2 x 2 heads of 64: 3.0 us, 4 rows: 2.1 us, of which a launch is 2.
struct AppendArgs {
  PoolView p;
  const bf16* qkv; long ldqkv;
  bf16* q; long ldq;
  const int* table; long ldt; int n_seq, cols;
  const int* seq; int rows_per_seq;
  const int* pos;
  long rows;
  int Hq, Hkv, rope_rows;
  const float *cos, *sin;
  int rows_per_block;
};

template <int D>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a) {
  constexpr int CH = D / 16;
  const int h0 = a.q ? 0 : a.Hq;
  const int items = (a.Hq + 2 * a.Hkv - h0) * CH;
  const long row0 = (long)blockIdx.x * a.rows_per_block;
  const int n = (int)min((long)a.rows_per_block, a.rows - row0) * items;
  for (int i = threadIdx.x; i < n; i += 256) {
    const int rl = i / items, it = i - rl * items;
    const long row = row0 + rl;
    const int c = it % CH, h = h0 + it / CH;
    const bf16* src = a.qkv + row * a.ldqkv + (long)h * D + 8 * c;
    bf16x8 x0 = *reinterpret_cast<const bf16x8*>(src), x1 = *reinterpret_cast<const bf16x8*>(src + D / 2);
    const int pos = a.pos[row];
    const long sq = a.seq ? (long)a.seq[row] : row / a.rows_per_seq;
    // a row that names no slot is padding: nothing of it is written
    if (pos < 0 || (pos >> a.p.shift) >= a.cols || sq < 0 || sq >= a.n_seq || (a.cos && pos >= a.rope_rows)) continue;
    const int page = a.table[sq * a.ldt + (pos >> a.p.shift)];
    if ((unsigned)page >= (unsigned)a.p.n_pages) continue;
    if (h < a.Hq + a.Hkv && a.cos) {
      const float* cs = a.cos + (long)pos * (D / 2) + 8 * c;
      const float* sn = a.sin + (long)pos * (D / 2) + 8 * c;
      const f32x4 c0 = *reinterpret_cast<const f32x4*>(cs), c1 = *reinterpret_cast<const f32x4*>(cs + 4);
      const f32x4 s0 = *reinterpret_cast<const f32x4*>(sn), s1 = *reinterpret_cast<const f32x4*>(sn + 4);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float cj = j < 4 ? c0[j & 3] : c1[j & 3], sj = j < 4 ? s0[j & 3] : s1[j & 3];
        const float u = (float)x0[j], w = (float)x1[j];
        x0[j] = (bf16)(u * cj - w * sj);
        x1[j] = (bf16)(w * cj + u * sj);
      }
    }
    bf16* dst;
    if (h < a.Hq) {
      dst = a.q + row * a.ldq + (long)h * D;
    } else {
      const bool isk = h < a.Hq + a.Hkv;
      const int kh = h - a.Hq - (isk ? 0 : a.Hkv);
      dst = (isk ? a.p.k : a.p.v) + (long)page * a.p.ps + (long)(pos & ((1 << a.p.shift) - 1)) * a.p.ss + kh * a.p.hs;
    }
    *reinterpret_cast<bf16x8*>(dst + 8 * c) = x0;
    *reinterpret_cast<bf16x8*>(dst + D / 2 + 8 * c) = x1;
  }
}

// ---- slx_prefix_attn -------------------------------------------------------------------------------------------
// o = sum_p e^{m_p - m} o_p / sum_p e^{m_p - m} l_p over the parts p of a row's keys, each with its own maximum m_p,
// sum l_p and unnormalised output o_p (the softmax is over the union, so any split of the keys is exact).
//
// The prefix of a group is read once for all of its width * n_q * (Hq / Hkv) query rows of a kv head; the sequences'
// own keys are workgroups of the same launch, with the n_q * (Hq / Hkv) rows of one sequence. A workgroup takes a tile
// of rows and one range of the keys and writes (m, l, o) of it; a second launch joins a row's parts.
//
// Per 32 keys and wave: S^T = K Q^T on v_mfma_f32_16x16x32_bf16 with the keys as rows and the queries as columns, so a
// lane holds 8 keys of ONE query, and the probabilities are already the B operand of O^T += V^T P^T (the sum over keys
// may take them in any order: slot j of lane group g is key 4g + j, or 16 + 4g + j - 4). V^T's A operand needs 8 keys
// of one d: a lane takes D/16 neighbouring d of each of its 8 keys and pairs them with v_perm_b32 (the MFMA row r of
// product e stands for d = (D/16) r + e). The row sums are one more MFMA, with an A operand of ones; a
// probability is two bf16 terms (softmax_step), so each product with P is two.
//
// Two forms of a workgroup, by the rows that share the keys:
//   direct (up to 8 rows of a prefix of 64-element heads, 16 of 128 or of own keys, 32 of a cache with pages of less than 8 slots): all 4
//     waves have the same rows; each takes every fourth 32-key tile straight into registers (K's next tile is requested once the
//     scores have used the last, V's after the output has), the waves' states are merged through LDS at the end. Few rows: the bytes
//     in flight count, and no wave waits for another. Many rows on such small pages cost twice the streamed form's time: 12 x 77
//     tokens on 640 keys 33 + 5 us on pages of 4 or 1, 15.6 on pages of 64.
//   streamed: 64 or 128 rows, so the keys are fetched once for all of them: tiles of 32 keys arrive by LDS-DMA in a ring, one
//     barrier a step. Rows of K and V lie in LDS with their 16-B chunks XOR-ed by the slot (and slots with bits 0 and 2
//     swapped), which keeps both operands' reads of 64 elements free of bank conflicts (of 128: 27 % of the LDS's cycles).
//     One page number for 8 keys (scalar load), so pages of at least 8 slots.
//
// Measured (main launch + join; 14 heads on 2 of 64 unless said). 2 x 16 sequences on 32771 shared and 300 .. 1000 own keys: 21.9 +
// 5.1 us, of which memory needs 8.5 (44 MB at 5.2 TB/s); VALU 26 % and MFMA 14 % of the SIMDs' cycles, the rest is the wait for the
// first tiles (5 us before and after the steps), the steps of few waves and uneven CUs (65 % of the CUs' cycles have a wave). 32 on 16411
// + 2000 of 32 heads on 8 of 128: 53.8 + 5.0 us, 215 MB = 3.7 TB/s. 8 x 8 on 1086: 7.6 + 3.1 us and 1 x 4 on 798: 5.9 + 2.5 us, where a
// launch takes 2 and the chain length -> page numbers -> keys -> merge the rest. Without a prefix, the whole call: one sequence of 839
// keys 8.1 us; 32 of 300 .. 1800 12.0, with 32 heads on 8 of 128 39.5 (137 MB, 3.5 TB/s); 16 of 8000 .. 16000 of those 177 (976 MB, 5.5 TB/s).
struct Seg {
  PoolView p;
  const int* tab; long ldt;
  const int* len;
  int cap;  // most keys a sequence of this segment has (host bound; the table's columns hold them)
  int ns;   // ranges a sequence's keys are split into at most
};
struct PAttnArgs {
  const bf16* q; long ldq;
  bf16* out; long ldo;
  float* lse;
  Seg pre, own;
  int W, Tq, Hq, Hkv, gq;
  unsigned gmul;  // r / gq = umulhi(r, gmul) (0: gq == 1)
  float c;        // scale * log2(e) > 0
  int mt_pre, mt_own;
  unsigned groups, n_pre;  // n_pre: workgroups of the prefix part
  int D;
  int direct;     // one part per row: the workgroups write the output themselves
  long R;         // rows * Hq
  float* ws;      // o [parts][R][D], then (m, l) [parts][R]
};

__host__ __device__ __forceinline__ int split_keys(int len, int ns) { return ((len + ns - 1) / ns + 127) & ~127; }
__device__ __forceinline__ int row_token(const PAttnArgs& a, int r) { return a.gmul ? (int)__umulhi((unsigned)r, a.gmul) : r; }

// one workgroup's share, uniform
struct Item {
  const bf16 *k, *v;  // of the kv head
  long ps, ss;
  int n_pages, shift;
  const int *tab, *lens;
  int cap, ns, range;
  int len, kb, ke;    // keys of the sequence; this range (item_range)
  bool causal;
  int kvh, ntok, mt, part;
  long tok0;          // first query token
};

__device__ __forceinline__ void item_segment(Item& w, const Seg& g, unsigned seq, bool causal) {
  w.ns = g.ns;
  w.cap = g.cap;
  w.causal = causal;
  w.k = g.p.k + w.kvh * g.p.hs;
  w.v = g.p.v + w.kvh * g.p.hs;
  w.ps = g.p.ps;
  w.ss = g.p.ss;
  w.n_pages = g.p.n_pages;
  w.shift = g.p.shift;
  w.tab = g.tab + seq * g.ldt;
  w.lens = g.len + seq;
}

template <int D, int NQ>
struct State {
  float m[NQ];
  f32x4 l[NQ], o[NQ][D / 16];
};

template <int D, int NQ>
__device__ __forceinline__ void state_init(State<D, NQ>& st) {
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    st.m[n] = -INFINITY;
    st.l[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < D / 16; ++e) st.o[n][e] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
}

// query rows r0 .. of a wave as B operands
template <int D, int NQ>
__device__ __forceinline__ void load_rows(const PAttnArgs& a, const Item& w, int r0, bf16x8 (&qf)[NQ][D / 32]) {
  const int col = threadIdx.x & 15, grp = (threadIdx.x & 63) >> 4, rows = w.ntok * a.gq;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int r = min(r0 + 16 * n + col, rows - 1), t = row_token(a, r);
    const bf16* qp = a.q + (w.tok0 + t) * a.ldq + (long)(w.kvh * a.gq + r - t * a.gq) * D + 8 * grp;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) qf[n][k] = *reinterpret_cast<const bf16x8*>(qp + 32 * k);
  }
}

// The item's range of keys, from the length on the device, while the queries are on their way. An empty range writes
// m = -inf for its rows (the join reads every part, and so does not wait for the lengths) and is done: false.
__device__ __forceinline__ bool item_range(const PAttnArgs& a, Item& w, int tile_rows) {
  w.len = max(0, min(*w.lens, w.cap));
  const int ks = split_keys(w.len, w.ns);
  w.kb = w.range * ks;
  w.ke = min(w.len, w.kb + ks);
  if (w.kb < w.len || a.direct) return true;
  const int r = w.mt * tile_rows + (int)threadIdx.x;
  if ((int)threadIdx.x < tile_rows && r < w.ntok * a.gq) {
    const int t = row_token(a, r);
    const long row = (w.tok0 + t) * a.Hq + w.kvh * a.gq + r - t * a.gq;
    float* ml = a.ws + (long)(a.pre.ns + a.own.ns) * a.R * a.D + ((long)w.part * a.R + row) * 2;
    *reinterpret_cast<float2*>(ml) = make_float2(-INFINITY, 0.f);
  }
  return false;
}

// the keys that each of a wave's rows sees
template <int NQ>
__device__ __forceinline__ void row_limits(const PAttnArgs& a, const Item& w, int r0, int (&lim)[NQ]) {
  const int col = threadIdx.x & 15, rows = w.ntok * a.gq;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int t = row_token(a, min(r0 + 16 * n + col, rows - 1));
    lim[n] = w.causal ? min(w.ke, w.len - a.Tq + t + 1) : w.ke;
  }
}

template <int D, int NQ>
__device__ __forceinline__ void scores(const bf16x8 (&kf)[2][D / 32], const bf16x8 (&qf)[NQ][D / 32], f32x4 (&s)[NQ][2]) {
#pragma unroll
  for (int n = 0; n < NQ; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      s[n][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < D / 32; ++k) s[n][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[h][k], qf[n][k], s[n][h], 0, 0, 0);
    }
}

// Scores of keys that are not there (dead: bit j of the lane's 8 keys) or that a row does not see (lim) to -inf.
template <int NQ>
__device__ __forceinline__ void mask_scores(f32x4 (&s)[NQ][2], unsigned dead, const int (&lim)[NQ], int k0) {
  const int grp = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int room = lim[n] - k0 - 4 * grp;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      s[n][j >> 2][j & 3] = (dead >> j & 1) | (16 * (j >> 2) + (j & 3) >= room) ? -INFINITY : s[n][j >> 2][j & 3];
  }
}

// Scores of T tiles to probabilities, with the state rescaled where a row's maximum has moved.
//
// A probability goes to the MFMA as two bf16 terms, p (1 + 2^-17) = hi + lo: hi its upper 16 bits as they are (so hi <= p), lo the rest,
// rounded (half a step of at most p 2^-7: 2^-15 p). One bf16 term alone is off by 2^-8 p and made the output's error up to 1.4 times
// that of its own rounding. The factor cancels in o / l; it keeps lo above 0, so that an infinite V keeps its sign in both products
// (0 * inf would be NaN). It costs a second product with V: 19.5 -> 22.1 us for 2 x 16 sequences on 32771 keys, 14.8 -> 16.2 for
// 12 x 77 tokens on 640, 45 -> 54 for 64 x 77; next to nothing where memory or latency bounds (57.8 -> 58.7 with the join for 32 on 16411
// keys of 8 heads of 128).
template <int D, int NQ, int T>
__device__ __forceinline__ void softmax_step(const f32x4 (&s)[T][NQ][2], float c, State<D, NQ>& st, bf16x8 (&ph)[T][NQ], bf16x8 (&pl)[T][NQ]) {
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    float mx = s[0][n][0][0];
#pragma unroll
    for (int j = 1; j < 8 * T; ++j) mx = fmaxf(mx, s[j >> 3][n][j >> 2 & 1][j & 3]);
    mx *= c;
    // the running maximum moves only when a score passes it by 2^8 (exact all the same: it cancels in o / l)
    if (__any(mx > st.m[n] + 8.0f)) {
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float mn = fmaxf(st.m[n], mx);
      const float r = st.m[n] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st.m[n] - mn);
      st.m[n] = mn;
      st.l[n] *= r;
#pragma unroll
      for (int e = 0; e < D / 16; ++e) st.o[n][e] *= r;
    }
    const float mu = st.m[n] == -INFINITY ? 0.f : st.m[n];
#pragma unroll
    for (int u = 0; u < T; ++u)
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        unsigned h[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][n][j >> 2][(j & 3) + i], c, -mu));
          h[i] = __float_as_uint(p) & 0xFFFF0000u;
          pl[u][n][j + i] = (bf16)__builtin_fmaf(p, 1.0f + 0x1p-17f, -__uint_as_float(h[i]));
        }
        union { unsigned u; bf16x2 b; } x;
        x.u = __builtin_amdgcn_perm(h[1], h[0], 0x07060302u);
        ph[u][n][j] = x.b[0];
        ph[u][n][j + 1] = x.b[1];
      }
  }
}

// Rows whose every score is NaN have no maximum but a sum that is NaN: a state like any other from here on, not an empty one.
template <int D, int NQ>
__device__ __forceinline__ void keep_nan(State<D, NQ>& st) {
#pragma unroll
  for (int n = 0; n < NQ; ++n) st.m[n] = st.l[n][0] != st.l[n][0] && st.m[n] == -INFINITY ? 0.f : st.m[n];
}

// V of keys that are not there becomes 0 (0 * NaN would reach every row); with `sift`, in a tile that some row of the wave does
// not see to its end, so do values that are not finite -> whether there were any (they are added at the end: add_nonfinite). A tile
// that every row sees keeps them: the product takes them to every row.
template <int D>
__device__ __forceinline__ bool clean_v(unsigned (&vr)[8][D / 32], unsigned dead, bool sift) {
  bool odd = false;
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      unsigned x = (dead >> j & 1) ? 0u : vr[j][i];
      if (sift) {
        const bool lo = (x & 0x7F80u) == 0x7F80u, hi = (x & 0x7F800000u) == 0x7F800000u;
        odd = odd || lo || hi;
        x = (lo ? 0u : (x & 0xFFFFu)) | (hi ? 0u : (x & 0xFFFF0000u));
      }
      vr[j][i] = x;
    }
  return odd;
}

template <int D, int NQ>
__device__ __forceinline__ void output_step(const unsigned (&vr)[8][D / 32], const bf16x8 (&ph)[NQ], const bf16x8 (&pl)[NQ], State<D, NQ>& st) {
  union { unsigned u[4]; bf16x8 b; } vt;
  vt.u[0] = vt.u[1] = vt.u[2] = vt.u[3] = 0x3F803F80u;  // ones
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    st.l[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt.b, ph[n], st.l[n], 0, 0, 0);
    st.l[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt.b, pl[n], st.l[n], 0, 0, 0);
  }
#pragma unroll
  for (int e = 0; e < D / 16; ++e) {
#pragma unroll
    for (int p = 0; p < 4; ++p)
      vt.u[p] = __builtin_amdgcn_perm(vr[2 * p + 1][e >> 1], vr[2 * p][e >> 1], (e & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      st.o[n][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt.b, ph[n], st.o[n][e], 0, 0, 0);
      st.o[n][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt.b, pl[n], st.o[n][e], 0, 0, 0);
    }
  }
}

__device__ __forceinline__ float natural_lse(float m, float l) {  // l sums p (1 + 2^-17)
  return m == -INFINITY ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f - 0x1p-17f;
}

// A row's (m, l, o) to the output or the workspace; a lane has d = (D/4) grp + (D/16) i + e of row r.
template <int D>
__device__ __forceinline__ void store_row(const PAttnArgs& a, const Item& w, int r, float m, float l, const f32x4 (&o)[D / 16]) {
  constexpr int NE = D / 16;
  const int grp = (threadIdx.x & 63) >> 4, t = row_token(a, r), head = w.kvh * a.gq + r - t * a.gq;
  const long row = (w.tok0 + t) * a.Hq + head;
  if (a.direct) {
    const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;  // no key seen: zeros
    bf16* op = a.out + (w.tok0 + t) * a.ldo + (long)head * D + (D / 4) * grp;
#pragma unroll
    for (int b = 0; b < NE / 2; ++b) {
      bf16x8 y;
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = (bf16)(o[(8 * b + j) % NE][(8 * b + j) / NE] * inv);
      *reinterpret_cast<bf16x8*>(op + 8 * b) = y;
    }
    if (a.lse && grp == 0) a.lse[row] = natural_lse(m, l);
  } else {
    float* op = a.ws + ((long)w.part * a.R + row) * D + (D / 4) * grp;
#pragma unroll
    for (int b = 0; b < NE; ++b) {
      f32x4 y;
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = o[(4 * b + j) % NE][(4 * b + j) / NE];
      *reinterpret_cast<f32x4*>(op + 4 * b) = y;
    }
    if (grp == 0) {
      float* ml = a.ws + (long)(a.pre.ns + a.own.ns) * a.R * D + ((long)w.part * a.R + row) * 2;
      *reinterpret_cast<float2*>(ml) = make_float2(m, l);
    }
  }
}

// Values that are not finite, of the keys from the 32 on that hold the first which some row does not see (no tile before is sifted):
// onto the rows that see them (p > 0 there, so inf and NaN arrive whatever p is; where a tile was not sifted they are there already and
// stay what they are), in what this thread has just stored. Rare, so kept small.
template <int D>
__device__ __forceinline__ void add_nonfinite(const PAttnArgs& a, const Item& w, int r) {
  const int grp = (threadIdx.x & 63) >> 4, t = row_token(a, r), head = w.kvh * a.gq + r - t * a.gq;
  const int from = max(w.kb, (max(0, w.len - a.Tq)) & ~31), to = min(w.ke, w.len - a.Tq + t + 1);
  bf16* op = a.out + (w.tok0 + t) * a.ldo + (long)head * D + (D / 4) * grp;
  float* wp = a.ws + ((long)w.part * a.R + (w.tok0 + t) * a.Hq + head) * D + (D / 4) * grp;
#pragma unroll 1
  for (int key = from; key < to; ++key) {
    const int e = w.tab[key >> w.shift];
    if ((unsigned)e >= (unsigned)w.n_pages) continue;
    const bf16* p = w.v + (long)e * w.ps + (long)(key & ((1 << w.shift) - 1)) * w.ss + (D / 4) * grp;
#pragma unroll 1
    for (int d = 0; d < D / 4; ++d) {
      const float v = (float)p[d];
      if (fabsf(v) < INFINITY) continue;
      if (a.direct) op[d] = (bf16)((float)op[d] + v);
      else wp[d] += v;
    }
  }
}

template <int D, int NQ>
__device__ __forceinline__ void attn_direct(const PAttnArgs& a, Item w, char* smem) {
  constexpr int KK = D / 32, NE = D / 16;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, grp = lane >> 4;
  const int rows = w.ntok * a.gq, r0 = w.mt * 16 * NQ;
  const int shift = w.shift, mask = (1 << shift) - 1;
  bf16x8 qf[NQ][KK];
  int lim[NQ];
  load_rows<D, NQ>(a, w, r0, qf);
  asm volatile("" ::: "memory");  // the queries are requested before the length is waited for
  if (!item_range(a, w, 16 * NQ)) return;
  row_limits<NQ>(a, w, r0, lim);
  // the causal edge of an own segment: token t of Tq sees keys <= len - Tq + t
  const int free_end = w.causal ? min(w.ke, w.len - a.Tq + row_token(a, r0) + 1) : w.ke;  // keys below it are seen by every row
  const int ke = w.causal ? min(w.ke, w.len - a.Tq + row_token(a, min(r0 + 16 * NQ, rows) - 1) + 1) : w.ke;
  const bf16 *kbase = w.k + 8 * grp, *vbase = w.v + NE * col;
  State<D, NQ> st;
  state_init(st);

  bf16x8 kf[2][KK];
  unsigned vr[8][NE / 2], bad = 0;  // bad: bit j = the lane's key j is on no page
  const bool fine = shift < 2;      // pages of 1 or 2 slots: a page number for each of a lane's keys
  auto entry = [&](int key) { return w.tab[min(key, w.len - 1) >> shift]; };
  auto at = [&](const bf16* base, int e, int key) {
    return base + ((unsigned)e < (unsigned)w.n_pages ? (long)e * w.ps : 0L) + (long)(key & mask) * w.ss;
  };
  auto ldv = [&](int j, const bf16* p) {
    if constexpr (NE == 4) {
      const u32x2 x = *reinterpret_cast<const u32x2*>(p);
      vr[j][0] = x[0]; vr[j][1] = x[1];
    } else {
      const u32x4 x = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
      for (int i = 0; i < NE / 2; ++i) vr[j][i] = x[i];
    }
  };
  int ek[2], ev[2];  // page numbers of the next tile to load
  auto entries_k = [&](int k0) {
#pragma unroll
    for (int s = 0; s < 2; ++s) ek[s] = entry(k0 + 16 * s + col);
  };
  auto entries_v = [&](int k0) {
    if (fine) return;
#pragma unroll
    for (int s = 0; s < 2; ++s) ev[s] = entry(k0 + 16 * s + 4 * grp);
  };
  auto load_k = [&](int k0) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const bf16* p = at(kbase, ek[s], k0 + 16 * s + col);
#pragma unroll
      for (int k = 0; k < KK; ++k) kf[s][k] = *reinterpret_cast<const bf16x8*>(p + 32 * k);
    }
  };
  auto load_v = [&](int k0) {
    bad = 0;
    if (fine) {
      int e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = entry(k0 + 16 * (j >> 2) + 4 * grp + (j & 3));
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        bad |= ((unsigned)e[j] >= (unsigned)w.n_pages ? 1u : 0u) << j;
        ldv(j, at(vbase, e[j], k0 + 4 * grp + (j & 3)));
      }
    } else {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        bad |= ((unsigned)ev[s] >= (unsigned)w.n_pages ? 15u : 0u) << (4 * s);
        const bf16* p = at(vbase, ev[s], k0 + 16 * s + 4 * grp);
#pragma unroll
        for (int j = 0; j < 4; ++j) ldv(4 * s + j, p + j * w.ss);
      }
    }
  };

  bool odd = false;
  int k0 = w.kb + 32 * wave;
  if (k0 < ke) {
    entries_k(k0);
    entries_v(k0);
    load_k(k0);
    load_v(k0);
    entries_k(k0 + 128);
    entries_v(k0 + 128);
  }
  for (; k0 < ke; k0 += 128) {
    f32x4 s[1][NQ][2];
    bf16x8 ph[1][NQ], pl[1][NQ];
    scores<D, NQ>(kf, qf, s[0]);
    const bool edge = k0 + 32 > free_end || __any(bad != 0);
    unsigned dead = bad;
    if (edge) {
      const int left = w.len - k0 - 4 * grp;
#pragma unroll
      for (int j = 0; j < 8; ++j) dead |= (16 * (j >> 2) + (j & 3) >= left ? 1u : 0u) << j;
      mask_scores<NQ>(s[0], dead, lim, k0);
    }
    const bool more = k0 + 128 < ke;
    if (more) {
      load_k(k0 + 128);
      entries_k(k0 + 256);
    }
    softmax_step<D, NQ, 1>(s, a.c, st, ph, pl);
    if (edge) odd = clean_v<D>(vr, dead, w.causal && a.Tq > 1 && k0 + 32 > free_end) || odd;
    output_step<D, NQ>(vr, ph[0], pl[0], st);
    if (more) {
      load_v(k0 + 128);
      entries_v(k0 + 256);
    }
  }

  // ---- the 4 waves' (m, l, o) into one: waves 2, 3 hand theirs to 0, 1, then 1 to 0
  float* sm = reinterpret_cast<float*>(smem);              // [4][16 NQ]
  float* sl = sm + 4 * 16 * NQ;                            // [4][16 NQ]
  f32x4* so = reinterpret_cast<f32x4*>(sl + 4 * 16 * NQ);  // [2][NQ * NE][64 lanes]
  float M[NQ], L[NQ];
  keep_nan(st);
  if (grp == 0) {
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      sm[wave * 16 * NQ + 16 * n + col] = st.m[n];
      sl[wave * 16 * NQ + 16 * n + col] = st.l[n][0];
    }
  }
  odd = __syncthreads_or(odd);
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    float mw[4];
#pragma unroll
    for (int v = 0; v < 4; ++v) mw[v] = sm[v * 16 * NQ + 16 * n + col];
    M[n] = fmaxf(fmaxf(mw[0], mw[1]), fmaxf(mw[2], mw[3]));
    L[n] = 0.f;
#pragma unroll
    for (int v = 0; v < 4; ++v)
      L[n] += mw[v] == -INFINITY ? 0.f : sl[v * 16 * NQ + 16 * n + col] * __builtin_amdgcn_exp2f(mw[v] - M[n]);
    const float r = st.m[n] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st.m[n] - M[n]);
#pragma unroll
    for (int e = 0; e < NE; ++e) st.o[n][e] *= r;
  }
  if (wave >= 2) {
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int e = 0; e < NE; ++e) so[((wave - 2) * NQ * NE + n * NE + e) * 64 + lane] = st.o[n][e];
  }
  __syncthreads();
  if (wave < 2) {
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int e = 0; e < NE; ++e) st.o[n][e] += so[(wave * NQ * NE + n * NE + e) * 64 + lane];
  }
  __syncthreads();
  if (wave == 1) {
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int e = 0; e < NE; ++e) so[(n * NE + e) * 64 + lane] = st.o[n][e];
  }
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int r = r0 + 16 * n + col;
    if (r >= rows) continue;
#pragma unroll
    for (int e = 0; e < NE; ++e) st.o[n][e] += so[(n * NE + e) * 64 + lane];
    store_row<D>(a, w, r, M[n], L[n], st.o[n]);
    if (odd) add_nonfinite<D>(a, w, r);
  }
}

template <int N>
__device__ __forceinline__ void wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
// this wave's pieces of the oldest tile are in LDS, with up to N younger tiles of PER pieces under way
template <int N, int PER>
__device__ __forceinline__ void wait_tiles(int younger) {
  if (younger >= N) wait_vm<N * PER>();
  else if constexpr (N > 0) wait_tiles<N - 1, PER>(younger);
}
// a barrier after this wave's LDS accesses alone, with its DMA still under way; no access moves across it
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
// 16 B a lane from base + off (bytes) to LDS at lds + 16 * lane
__device__ __forceinline__ void dma16(const void* base, unsigned off, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory", "m0");
}

// A streamed workgroup: NW waves, RV of them side by side over RW rows, and as many teams as that leaves, each of which takes tiles
// of its own of every step of the ring, T tiles of 32 keys; the teams are joined at the end. With two teams of 64 rows of 64 elements
// an operand read from LDS serves 32 rows of a wave instead of 16: 24.4 us instead of 25.0 for 340 whole-row tiles; a range of
// 128 keys is over before that pays for the join of the teams: 6.7 us instead of 6.0 for 4 sequences on 798 keys.
template <int D, int RW, int NW, int RV>
struct Shape {
  static constexpr int RWV = RV, NQ = RW / 16 / RWV, TEAMS = NW / RWV;
  static constexpr int T = TEAMS > 1 ? TEAMS : D == 64 ? 2 : 1, UW = T / TEAMS;  // tiles a step, and of them a team's
  static constexpr int SLOTS = D == 128 && T == 1 ? 4 : 3;
  static constexpr int LDS = SLOTS * (T * 2 * 32 * D * 2 + 4 * T);
};

// The keys of one segment into the state of a wave's rows r0 .. (the workgroup's from rw); whether values were sifted out.
// The LDS is free when it is called, and its last tiles may still be read when it returns.
template <int D, int RW, int NW, int RV>
__device__ __forceinline__ bool stream_keys(const PAttnArgs& a, const Item& w, int rw, int r0,
                                            const bf16x8 (&qf)[Shape<D, RW, NW, RV>::NQ][D / 32], State<D, Shape<D, RW, NW, RV>::NQ>& st, char* smem) {
  typedef Shape<D, RW, NW, RV> S;
  constexpr int KK = D / 32, NE = D / 16, CH = D / 8, TILE = 32 * D * 2, T = S::T, SLOTS = S::SLOTS, STEP = 32 * T, NQ = S::NQ, UW = S::UW;
  constexpr int TI = 4 * T / NW;       // tiles of a step that a wave brings 8 keys of
  constexpr int PER = TI * 2 * D / 64;  // DMA pieces a wave and step
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, grp = lane >> 4;
  const int wk = 8 * (wave & 3), wt = wave >> 2;  // its 8 keys of a tile, and which tile of each NW / 4
  const int rows = w.ntok * a.gq, shift = w.shift, mask = (1 << shift) - 1;
  unsigned char* badb = reinterpret_cast<unsigned char*>(smem + SLOTS * T * 2 * TILE);  // [SLOTS][T][4]: 8 keys a wave, 0 or 255
  const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)LDS_PTR(char, smem));
  int lim[NQ];
  row_limits<NQ>(a, w, r0, lim);
  auto tok_of = [&](int r) { return row_token(a, min(r, rows - 1)); };
  const int free_end = w.causal ? min(w.ke, w.len - a.Tq + tok_of(r0) + 1) : w.ke;  // seen by every row of the wave
  const int ke = w.causal ? min(w.ke, w.len - a.Tq + tok_of(rw + RW - 1) + 1) : w.ke;
  const int kw = r0 >= rows ? 0 : w.causal ? min(w.ke, w.len - a.Tq + tok_of(r0 + 16 * NQ - 1) + 1) : w.ke;  // this wave's last
  const int nt = ke > w.kb ? (ke - w.kb + STEP - 1) / STEP : 0;
  // LDS rows: slot of key x = x with bits 0 and 2 swapped; chunk c of a slot lies at c ^ swz(slot)
  auto slot_of = [](int x) { return (x & ~5) | (x & 1) << 2 | (x >> 2 & 1); };
  auto swz = [](int slot) { return D == 64 ? slot >> 1 & 7 : slot & 15; };
  typedef const int __attribute__((address_space(4))) cint;
  auto entry = [&](int t, int u) {  // the page of this wave's 8 keys of its tile u of step t
    const int key = min(w.kb + STEP * min(t, nt - 1) + 32 * (u * (NW / 4) + wt) + wk, w.len - 1);
    return ((cint*)(uintptr_t)w.tab)[__builtin_amdgcn_readfirstlane(key >> shift)];
  };
  // A piece is 1 KiB: the wave's 8 keys lie on one page, so its address is a scalar and the lane's place among them.
  unsigned off[PER / (2 * TI)];
#pragma unroll
  for (int i = 0; i < PER / (2 * TI); ++i) {
    const int slot = wk + (64 / CH) * i + lane / CH;
    off[i] = 2u * ((unsigned)(slot_of(slot) & 7) * (unsigned)w.ss + 8u * (unsigned)((lane % CH) ^ swz(slot)));
  }
  auto issue = [&](int t, const int (&e)[TI]) {
#pragma unroll
    for (int u = 0; u < TI; ++u) {
      const int tile = u * (NW / 4) + wt, at = (t % SLOTS) * T + tile;
      const bool ok = (unsigned)e[u] < (unsigned)w.n_pages;
      const long from = (ok ? (long)e[u] * w.ps : 0L) + (long)((w.kb + STEP * t + 32 * tile + wk) & mask) * w.ss;
      if (lane == 0) badb[at * 4 + (wave & 3)] = ok ? 0 : 255;
#pragma unroll
      for (int i = 0; i < PER / (2 * TI); ++i) {
        const unsigned to = lds0 + at * 2 * TILE + (wk + (64 / CH) * i) * D * 2;
        dma16(w.k + from, off[i], to);
        dma16(w.v + from, off[i], to + TILE);
      }
    }
  };
  int en[TI];
  if (nt > 0) {
    int e[SLOTS - 1][TI];
#pragma unroll
    for (int i = 0; i < SLOTS - 1; ++i)
#pragma unroll
      for (int u = 0; u < TI; ++u) e[i][u] = entry(i, u);
#pragma unroll
    for (int u = 0; u < TI; ++u) en[u] = entry(SLOTS - 1, u);
#pragma unroll
    for (int i = 0; i < SLOTS - 1; ++i)
      if (i < nt) issue(i, e[i]);
  }
  int ko[KK], vo[8];  // this lane's operands within a tile
#pragma unroll
  for (int k = 0; k < KK; ++k) ko[k] = slot_of(col) * D * 2 + ((4 * k + grp) ^ swz(slot_of(col))) * 16;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int slot = slot_of(16 * (j >> 2) + 4 * grp + (j & 3));
    vo[j] = TILE + slot * D * 2 + (NE == 4 ? ((col >> 1) ^ swz(slot)) * 16 + (col & 1) * 8 : (col ^ swz(slot)) * 16);
  }
  bool odd = false;
  for (int t = 0; t < nt; ++t) {
    const int k0 = w.kb + STEP * t;
    wait_tiles<SLOTS - 2, PER>(nt - 1 - t);
    lds_barrier();  // every wave has read the slot that is filled next
    if (t + SLOTS - 1 < nt) {
      issue(t + SLOTS - 1, en);
#pragma unroll
      for (int u = 0; u < TI; ++u) en[u] = entry(t + SLOTS, u);
    }
    const int u0 = wave / S::RWV * UW;
    if (k0 + 32 * u0 >= kw) continue;
    f32x4 s[UW][NQ][2];
    bf16x8 ph[UW][NQ], pl[UW][NQ];
    unsigned vr[UW][8][NE / 2], bads[UW], dead[UW];
#pragma unroll
    for (int v = 0; v < UW; ++v) {
      const char* tile = smem + ((t % SLOTS) * T + u0 + v) * 2 * TILE;
      bads[v] = *reinterpret_cast<const unsigned*>(badb + ((t % SLOTS) * T + u0 + v) * 4);
      bf16x8 kf[2][KK];
#pragma unroll
      for (int k = 0; k < KK; ++k) {  // keys 16 apart lie 16 slots apart, under the same swizzle
        kf[0][k] = *reinterpret_cast<const bf16x8*>(tile + ko[k]);
        kf[1][k] = *reinterpret_cast<const bf16x8*>(tile + ko[k] + 16 * D * 2);
      }
      scores<D, NQ>(kf, qf, s[v]);
    }
#pragma unroll
    for (int v = 0; v < UW; ++v) {
      const char* tile = smem + ((t % SLOTS) * T + u0 + v) * 2 * TILE;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (NE == 4) {
          const u32x2 x = *reinterpret_cast<const u32x2*>(tile + vo[j]);
          vr[v][j][0] = x[0]; vr[v][j][1] = x[1];
        } else {
          const u32x4 x = *reinterpret_cast<const u32x4*>(tile + vo[j]);
#pragma unroll
          for (int i = 0; i < NE / 2; ++i) vr[v][j][i] = x[i];
        }
      }
    }
    unsigned any_bad = 0;
#pragma unroll
    for (int v = 0; v < UW; ++v) any_bad |= bads[v];
    const bool edge = k0 + 32 * (u0 + UW) > free_end || __builtin_amdgcn_readfirstlane(any_bad) != 0;
    if (edge) {
#pragma unroll
      for (int v = 0; v < UW; ++v) {
        const int kv = k0 + 32 * (u0 + v);
        dead[v] = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int x = 16 * (j >> 2) + 4 * grp + (j & 3);
          dead[v] |= (kv + x >= w.len || (bads[v] >> x & 1) ? 1u : 0u) << j;
        }
        mask_scores<NQ>(s[v], dead[v], lim, kv);
      }
    }
    softmax_step<D, NQ, UW>(s, a.c, st, ph, pl);
    if (edge) {
#pragma unroll
      for (int v = 0; v < UW; ++v) odd = clean_v<D>(vr[v], dead[v], w.causal && a.Tq > 1 && k0 + 32 * (u0 + v + 1) > free_end) || odd;
    }
#pragma unroll
    for (int v = 0; v < UW; ++v) output_step<D, NQ>(vr[v], ph[v], pl[v], st);
  }
  return odd;
}

// the queries are here before the first DMA is counted
template <int D, int NQ>
__device__ __forceinline__ void settle_rows(bf16x8 (&qf)[NQ][D / 32]) {
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
#pragma unroll
  for (int n = 0; n < NQ; ++n)
#pragma unroll
    for (int k = 0; k < D / 32; ++k) asm volatile("" : "+v"(qf[n][k]));
}

template <int D, int RW, int NW, int RV>
__device__ __forceinline__ void store_stream(const PAttnArgs& a, const Item& w, int r0, bool odd, State<D, Shape<D, RW, NW, RV>::NQ>& st,
                                             char* smem) {
  typedef Shape<D, RW, NW, RV> S;
  constexpr int NQ = S::NQ, NE = D / 16, HAND = NQ * (NE + 1) * 64;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15;
  odd = __any(odd);
  keep_nan(st);
  if constexpr (S::TEAMS > 1) {
    static_assert((NW - S::RWV) * HAND * 16 <= S::LDS, "the teams' states take the ring's place");
    f32x4* so = reinterpret_cast<f32x4*>(smem);  // [team 1 ..][rows' wave][NQ][NE + 1][lane]
    __syncthreads();
    if (wave >= S::RWV) {
      f32x4* to = so + (wave - S::RWV) * HAND + lane;
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
#pragma unroll
        for (int e = 0; e < NE; ++e) to[(n * (NE + 1) + e) * 64] = st.o[n][e];
        to[(n * (NE + 1) + NE) * 64] = f32x4{st.m[n], st.l[n][0], odd ? 1.f : 0.f, 0.f};
      }
    }
    __syncthreads();
    if (wave >= S::RWV) return;
#pragma unroll
    for (int k = 0; k < S::TEAMS - 1; ++k) {
      const f32x4* from = so + (k * S::RWV + wave) * HAND + lane;
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const f32x4 x = from[(n * (NE + 1) + NE) * 64];
        const float M = fmaxf(st.m[n], x[0]);
        const float r0_ = st.m[n] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st.m[n] - M);
        const float r1_ = x[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x[0] - M);
        st.l[n][0] = st.l[n][0] * r0_ + x[1] * r1_;
        st.m[n] = M;
        odd = odd || x[2] != 0.f;
#pragma unroll
        for (int e = 0; e < NE; ++e) st.o[n][e] = st.o[n][e] * r0_ + from[(n * (NE + 1) + e) * 64] * r1_;
      }
    }
    odd = __any(odd);
  }
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int r = r0 + 16 * n + col;
    if (r >= w.ntok * a.gq) continue;
    store_row<D>(a, w, r, st.m[n], st.l[n][0], st.o[n]);
    if (odd) add_nonfinite<D>(a, w, r);
  }
}

template <int D, int RW, int NW, int RV>
__device__ __forceinline__ int wave_row(int rw) {  // a wave's first row
  typedef Shape<D, RW, NW, RV> S;
  return rw + (__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % S::RWV) * 16 * S::NQ;
}

template <int D, int RW, int NW, int RV>
__device__ __forceinline__ void attn_stream(const PAttnArgs& a, Item w, char* smem) {
  constexpr int NQ = Shape<D, RW, NW, RV>::NQ;
  const int rw = w.mt * RW, r0 = wave_row<D, RW, NW, RV>(rw);
  bf16x8 qf[NQ][D / 32];
  load_rows<D, NQ>(a, w, r0, qf);
  asm volatile("" ::: "memory");  // the queries are requested before the length is waited for
  if (!item_range(a, w, RW)) return;
  State<D, NQ> st;
  state_init(st);
  settle_rows<D, NQ>(qf);
  const bool odd = stream_keys<D, RW, NW, RV>(a, w, rw, r0, qf, st, smem);
  store_stream<D, RW, NW, RV>(a, w, r0, odd, st, smem);
}

// kinds of a workgroup: direct with 16 or 32 rows, streamed with 64 or 128
enum { kD16 = 0, kD32 = 1, kS64 = 2, kS128 = 3 };
constexpr int kKindRows[4] = {16, 32, 64, 128};
template <int D, int KIND>
__device__ __forceinline__ void attn_kind(const PAttnArgs& a, const Item& w, char* smem) {
  if constexpr (KIND == kD16) attn_direct<D, 1>(a, w, smem);
  else if constexpr (KIND == kD32) attn_direct<D, 2>(a, w, smem);
  else if constexpr (KIND == kS64) attn_stream<D, 64, 4, 4>(a, w, smem);
  else attn_stream<D, 128, 4, 4>(a, w, smem);
}
template <int D>
constexpr int kind_lds(int kind) {
  return kind == kS64 ? Shape<D, 64, 4, 4>::LDS : kind == kS128 ? Shape<D, 128, 4, 4>::LDS : 2 * 4 * 16 * (kind + 1) * 4 + 2 * (kind + 1) * (D / 16) * 64 * 16;
}

template <int D, int KP, int KO>
__global__ __launch_bounds__(256, 2) void prefix_attn_kernel(PAttnArgs a) {
  constexpr int LDS = kind_lds<D>(KP) > kind_lds<D>(KO) ? kind_lds<D>(KP) : kind_lds<D>(KO);
  __shared__ __attribute__((aligned(16))) char smem[LDS];
  unsigned b = blockIdx.x;
  const bool pre = b < a.n_pre;
  Item w;
  unsigned seq;
  if (pre) {  // [group][kv head][range][row tile]; 8 neighbours stay 8 apart, so the row tiles of a range share an XCD's L2
    const unsigned x = b & 7, y = b >> 3;
    w.mt = (int)(y % (unsigned)a.mt_pre);
    b = (y / (unsigned)a.mt_pre) * 8 + x;
    w.part = (int)(b % (unsigned)a.pre.ns);
    b /= (unsigned)a.pre.ns;
    w.kvh = (int)(b % (unsigned)a.Hkv);
    seq = b / (unsigned)a.Hkv;
    if (seq >= a.groups) return;  // the grid is padded to a multiple of 8
    w.tok0 = (long)seq * a.W * a.Tq;
    w.ntok = a.W * a.Tq;
  } else {  // [sequence][row tile][kv head][range]
    b -= a.n_pre;
    w.part = (int)(b % (unsigned)a.own.ns);
    b /= (unsigned)a.own.ns;
    w.kvh = (int)(b % (unsigned)a.Hkv);
    b /= (unsigned)a.Hkv;
    w.mt = (int)(b % (unsigned)a.mt_own);
    seq = b / (unsigned)a.mt_own;
    w.tok0 = (long)seq * a.Tq;
    w.ntok = a.Tq;
  }
  w.range = w.part;
  item_segment(w, pre ? a.pre : a.own, seq, !pre);
  if (!pre) w.part += a.pre.ns;
  if constexpr (KP == KO) {
    attn_kind<D, KP>(a, w, smem);
  } else {
    if (pre) attn_kind<D, KP>(a, w, smem);
    else attn_kind<D, KO>(a, w, smem);
  }
}

// Many new tokens in many sequences: a workgroup takes 64 or 128 rows of ONE sequence through the prefix and then its own
// keys, so there are no parts to write and join (the prefix is fetched again for every tile of rows, from L2).
template <int D, int RW, int NW, int RV>
__global__ __launch_bounds__(64 * NW, 2) void prefix_attn_whole_kernel(PAttnArgs a) {
  constexpr int NQ = Shape<D, RW, NW, RV>::NQ;
  __shared__ __attribute__((aligned(16))) char smem[Shape<D, RW, NW, RV>::LDS];
  unsigned b = blockIdx.x;  // [kv head][sequence][row tile]: neighbours share the prefix
  Item w;
  w.mt = (int)(b % (unsigned)a.mt_own);
  b /= (unsigned)a.mt_own;
  const unsigned n = a.groups * (unsigned)a.W, seq = b % n;
  w.kvh = (int)(b / n);
  w.tok0 = (long)seq * a.Tq;
  w.ntok = a.Tq;
  w.range = w.part = 0;
  const int rw = w.mt * RW, r0 = wave_row<D, RW, NW, RV>(rw);
  bf16x8 qf[NQ][D / 32];
  load_rows<D, NQ>(a, w, r0, qf);
  asm volatile("" ::: "memory");  // the queries are requested before the lengths are waited for
  item_segment(w, a.pre, seq / (unsigned)a.W, false);
  item_range(a, w, RW);
  State<D, NQ> st;
  state_init(st);
  settle_rows<D, NQ>(qf);
  stream_keys<D, RW, NW, RV>(a, w, rw, r0, qf, st, smem);
  item_segment(w, a.own, seq, true);
  item_range(a, w, RW);
  lds_barrier();  // the ring is free when every wave has read the prefix's last tiles
  const bool odd = stream_keys<D, RW, NW, RV>(a, w, rw, r0, qf, st, smem);
  store_stream<D, RW, NW, RV>(a, w, r0, odd, st, smem);
}

// Joins the parts of a row: D / 4 threads, four d each, times PG groups that share the parts out, B at a time: up to 8 parts at
// once by one group, up to 16 by four, more by a whole workgroup, so that the loads of a row make few rounds. 8 parts of 56 rows:
// 2.4 us by one group, 3.3 by four; 11 parts of 896 rows: 3.1 by four, 4.0 by one, 4.3 by the workgroup; 22 parts of 1024 rows of 128:
// 4.9 (12 MB, 2.4 TB/s).
template <int D, int PG, int B>
__global__ __launch_bounds__(256) void prefix_attn_join_kernel(PAttnArgs a) {
  constexpr int TPR = D / 4, RPB = 256 / (TPR * PG);
  __shared__ float sml[RPB][PG][2];
  __shared__ __attribute__((aligned(16))) f32x4 so[RPB][PG][TPR];
  const int d4 = threadIdx.x % TPR, pg = threadIdx.x / TPR % PG, rl = threadIdx.x / (TPR * PG), parts = a.pre.ns + a.own.ns;
  const bool off = (long)blockIdx.x * RPB + rl >= a.R;  // behind the last row: along with it up to the barrier
  const long row = min((long)blockIdx.x * RPB + rl, a.R - 1);
  const float2* ml = reinterpret_cast<const float2*>(a.ws + parts * a.R * D) + row;
  const float* ob = a.ws + row * D + 4 * d4;
  float m = -INFINITY, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](const float (&xm)[B], const float (&xl)[B], const f32x4 (&y)[B]) {
    float mn = m;
#pragma unroll
    for (int u = 0; u < B; ++u) mn = fmaxf(mn, xm[u]);
    const float r = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
    l *= r;
    o *= r;
#pragma unroll
    for (int u = 0; u < B; ++u) {
      if (xm[u] == -INFINITY) continue;  // its o was not computed from any key
      const float w = __builtin_amdgcn_exp2f(xm[u] - mn);
      l = __builtin_fmaf(w, xl[u], l);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = __builtin_fmaf(w, y[u][j], o[j]);
    }
    m = mn;
  };
  for (int i0 = pg; i0 < parts; i0 += B * PG) {
    float xm[B], xl[B];
    f32x4 y[B];
#pragma unroll
    for (int u = 0; u < B; ++u) {
      const int p = min(i0 + u * PG, parts - 1);
      const float2 x = ml[(long)p * a.R];
      y[u] = *reinterpret_cast<const f32x4*>(ob + (long)p * a.R * D);
      xm[u] = i0 + u * PG < parts ? x.x : -INFINITY;
      xl[u] = x.y;
    }
    add(xm, xl, y);
  }
  if constexpr (PG > 1) {
    so[rl][pg][d4] = o;
    if (d4 == 0) { sml[rl][pg][0] = m; sml[rl][pg][1] = l; }
    __syncthreads();
    if (pg) return;
    m = -INFINITY;
    l = 0.f;
    o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i0 = 0; i0 < PG; i0 += B) {
      float xm[B], xl[B];
      f32x4 y[B];
#pragma unroll
      for (int u = 0; u < B; ++u) { xm[u] = sml[rl][i0 + u][0]; xl[u] = sml[rl][i0 + u][1]; y[u] = so[rl][i0 + u][d4]; }
      add(xm, xl, y);
    }
  }
  if (off) return;
  const long tok = row / a.Hq;
  const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
  bf16x4 y;
#pragma unroll
  for (int j = 0; j < 4; ++j) y[j] = (bf16)(o[j] * inv);
  *reinterpret_cast<bf16x4*>(a.out + tok * a.ldo + (row - tok * a.Hq) * D + 4 * d4) = y;
  if (a.lse && d4 == 0) a.lse[row] = natural_lse(m, l);
}

// Row tiles and key ranges of a call: a rule on sizes, page sizes and the host's bounds alone, so a captured call replays
// for any lengths up to them. As many ranges as give about kTarget workgroups, each of at least 128 keys; or whole rows.
//
// Whole rows, a tile of 64 rows of one sequence through the prefix and its own keys, write no parts and need no join, but fetch the
// prefix for every tile and run alone (1.5 us for 128 keys of 64 elements on an 8-wave workgroup, 3 us of 128). Measured against
// parts + join (us; 14 heads on 2 of 64 unless said):
//   12 sequences of 77 tokens:   640 shared keys 16.2, 28.3 + 5.3;  1800: 30.8, 36.4 + 5.3;  8000: 100, 83 + 6
//   10 of 60 (140 tiles), 1280:  22.4, 24.2 + 6.3   4 of 40 (40 tiles), 640: 14.6, 10.8 + 3.9       1 of 3 (2 tiles), 200: 10.4, 6.8 + 2.0
//   32 heads on 8 of 128:        8 of 64 (256 tiles), 1280: 37, 45 + 9   4 of 40 (96), 640: 19.7, 19.7 + 4.8   4 of 40, 1280: 30.1, 23.2 + 7.5
// Ranges: 512 / 768 / 1024 / 1536 workgroups for 2 x 16 sequences on 32771 keys 24.4 + 4.9 / 22.0 + 5.1 / 23.3 + 6.2 / 23.4 + 6.2, for 32
// on 16411 keys of 8 heads of 128 64.8 + 4.7 / 54.8 + 4.9 / 53.8 + 5.3 / 61.0 + 6.9.
constexpr long kTarget = 768, kCUs = 256;
struct PAttnPlan { int kp, ko, mtp, mto, nsp, nso, whole; };  // whole: waves of a workgroup, or 0
// the most units of 128 keys that tiles of whole rows run through
static long whole_units(int D, long tiles) { return tiles >= (D == 64 ? 64 : 192) ? 12 : tiles >= (D == 64 ? 16 : 64) ? 7 : 0; }
static PAttnPlan plan_attn(const slx_prefix_attn_desc* d, int capp, int capo) {
  PAttnPlan p;
  const int gq = d->Hq / d->own_pool.heads;
  auto kind = [](long rows, const slx_kv_pool& pool, long direct) {
    // Streamed tiles: one page number for 8 keys, whose offsets on the page fit 32 bits. Direct / streamed prefixes, us of the main
    // launch: 7 rows on 798 keys 5.7 / 5.7, on 32771 7.8 / 7.3 (5.2 / 5.3 of them joined); 14 rows 5.8 / 5.8 and 8.4 / 8.2; 28 rows
    // 7.0 / 6.0 and 11.8 / 9.8. Heads of 128: 12 rows on 16411 17.6 / 18.7, 16 rows on 4 x 16411 60.3 / 59.7, 32 rows on 16411
    // 23.5 / 20.5. Own keys, many short sequences of 7 rows beside the prefix: 21.8 / 25.2 (2 x 16 on 32771) and 8.5 / 20.8 (8 x 8 on
    // 1086). 64 / 128 rows a tile: 112 rows on 32771 keys 21.5 / 21.9, on 1086 6.7 / 7.9; heads of 128, 128 rows on 16411 58.8 / 53.8
    // (the keys pass through L2 once instead of twice).
    const bool streams = pool.page >= 8 && pool.slot_stride < (1 << 27);
    return rows <= (streams ? direct : 16) ? kD16 : !streams ? kD32 : rows <= 64 ? kS64 : kS128;
  };
  const long rp = (long)d->width * d->n_q * gq, ro = (long)d->n_q * gq, heads = d->own_pool.heads;
  const long seqs = (long)d->groups * d->width * heads, t64 = (ro + 63) / 64, t128 = (ro + 127) / 128;
  const long up = (capp + 127) / 128, uo = (capo + 127) / 128;  // units of 128 keys
  p.whole = 0;
  p.ko = kind(ro, d->own_pool, 16);
  p.kp = capp > 0 ? kind(rp, d->prefix_pool, d->own_pool.head_dim == 64 ? 8 : 16) : p.ko;
  if (capp > 0 && p.kp >= kS64 && p.ko >= kS64 && up + uo <= whole_units(d->own_pool.head_dim, seqs * t64)) {
    p.ko = p.kp = 2 * seqs * t128 >= 3 * kCUs ? kS128 : kS64;
    p.whole = p.ko == kS64 && seqs * t64 <= kCUs ? 8 : 4;  // one workgroup a CU: 8 waves (16.2 us above, 4 waves 19.0); two of them: 4 (340 tiles: 24.6, 30.4)
    p.mto = p.mtp = (int)(p.ko == kS128 ? t128 : t64);
    p.nsp = p.nso = 1;
    return p;
  }
  if (p.kp == kD32 && p.ko >= kS64) p.ko = kD32;       // fewer kernels: a streamed own part goes with a streamed prefix,
  if (p.kp == kS128 && p.ko == kS64) p.ko = kS128;     // of the same rows
  p.mtp = (int)((rp + kKindRows[p.kp] - 1) / kKindRows[p.kp]);
  p.mto = (int)((ro + kKindRows[p.ko] - 1) / kKindRows[p.ko]);
  const long ip = d->groups * heads * p.mtp, io = seqs * p.mto;
  const long per = (ip * up + io * uo + kTarget - 1) / kTarget, u = per > 1 ? per : 1;
  p.nsp = (int)((up + u - 1) / u);
  p.nso = (int)((uo + u - 1) / u);
  if (p.nso < 1) p.nso = 1;
  return p;
}
static bool is_direct(const PAttnPlan& p) { return p.whole || p.nsp + p.nso == 1; }

static int check_pool(const slx_kv_pool& p, const char* who) {
  SLX_CHECK_ARG(p.k && p.v && ((uintptr_t)p.k & 15) == 0 && ((uintptr_t)p.v & 15) == 0, "%s: k and v must be 16-B aligned", who);
  SLX_CHECK_ARG(p.head_dim == 64 || p.head_dim == 128, "%s: head_dim must be 64 or 128 (got %d)", who, p.head_dim);
  SLX_CHECK_ARG(p.heads > 0 && p.n_pages > 0 && log2_exact(p.page) >= 0, "%s: heads, n_pages > 0 and page a power of two", who);
  SLX_CHECK_ARG(p.page_stride % 8 == 0 && p.slot_stride % 8 == 0 && p.head_stride % 8 == 0 && p.page_stride >= 0 &&
                p.slot_stride >= 0 && p.head_stride >= 0, "%s: pool strides must be multiples of 8 elements", who);
  return 0;
}
static PoolView view(const slx_kv_pool& p) {
  return PoolView{(bf16*)p.k, (bf16*)p.v, (long)p.page_stride, (long)p.slot_stride, (long)p.head_stride, p.n_pages, log2_exact(p.page)};
}
static int cap_of(int most, int cols, int page) {  // keys that the bound and the table's columns allow
  const long c = (long)cols * page;
  return most < c ? most : (int)c;
}

static int check_attn(const slx_prefix_attn_desc* d, int* capp, int* capo) {
  SLX_CHECK_ARG(d != nullptr, "slx_prefix_attn: null desc");
  if (int rc = check_pool(d->own_pool, "slx_prefix_attn")) return rc;
  SLX_CHECK_ARG(d->groups >= 0 && d->width > 0 && d->n_q > 0 && d->Hq > 0 && d->Hq % d->own_pool.heads == 0,
                "slx_prefix_attn: groups >= 0, width, n_q > 0 and Hq a multiple of the pool's heads");
  SLX_CHECK_ARG((double)d->groups * d->width * d->n_q * d->Hq < 2147483648.0, "slx_prefix_attn: too many rows");
  // row / gq is a multiplication (exact while row * gq < 2^32)
  SLX_CHECK_ARG((double)d->width * d->n_q * (d->Hq / d->own_pool.heads) * (d->Hq / d->own_pool.heads) < 4294967296.0,
                "slx_prefix_attn: too many rows");
  SLX_CHECK_ARG(d->scale > 0.0f && d->scale * 1.44269504088896341f < INFINITY, "slx_prefix_attn: scale must be positive and, times log2(e), finite");
  SLX_CHECK_ARG(d->max_own >= 0 && d->ocols > 0 && d->ldot >= d->ocols, "slx_prefix_attn: max_own >= 0, ldot >= ocols > 0");
  *capo = cap_of(d->max_own, d->ocols, d->own_pool.page);
  *capp = 0;
  if (d->ptab) {
    if (int rc = check_pool(d->prefix_pool, "slx_prefix_attn (prefix)")) return rc;
    SLX_CHECK_ARG(d->prefix_pool.heads == d->own_pool.heads && d->prefix_pool.head_dim == d->own_pool.head_dim,
                  "slx_prefix_attn: the two pools differ in heads or head_dim");
    SLX_CHECK_ARG(d->plen && d->max_prefix >= 0 && d->pcols > 0 && d->ldpt >= d->pcols,
                  "slx_prefix_attn: a prefix needs plen, max_prefix >= 0, ldpt >= pcols > 0");
    *capp = cap_of(d->max_prefix, d->pcols, d->prefix_pool.page);
  }
  SLX_CHECK_ARG(*capo <= 1 << 30 && *capp <= 1 << 30, "slx_prefix_attn: max_own and max_prefix (or the tables' columns) must be <= 2^30 keys");
  return 0;
}

template <int D>
static bool launch_attn(const PAttnPlan& p, dim3 grid, hipStream_t st, const PAttnArgs& a) {
  if (p.whole) {
    if (p.ko == kS128) hipLaunchKernelGGL((prefix_attn_whole_kernel<D, 128, 4, 4>), grid, dim3(256), 0, st, a);
    else if (p.whole == 8) hipLaunchKernelGGL((prefix_attn_whole_kernel<D, 64, 8, D == 64 ? 2 : 4>), grid, dim3(512), 0, st, a);
    else hipLaunchKernelGGL((prefix_attn_whole_kernel<D, 64, 4, D == 64 ? 2 : 4>), grid, dim3(256), 0, st, a);
    return true;
  }
#define SLX_PA(P, O)                                                                                         \
  if (p.kp == P && p.ko == O) {                                                                              \
    hipLaunchKernelGGL((prefix_attn_kernel<D, P, O>), grid, dim3(256), 0, st, a);                            \
    return true;                                                                                             \
  }
  SLX_PA(kD16, kD16) SLX_PA(kD32, kD16) SLX_PA(kD32, kD32) SLX_PA(kS64, kD16) SLX_PA(kS64, kD32) SLX_PA(kS64, kS64)
  SLX_PA(kS128, kD16) SLX_PA(kS128, kD32) SLX_PA(kS128, kS128)
#undef SLX_PA
  return false;
}
static int join_groups(int D, int parts) { return parts <= 8 ? 1 : parts <= 16 ? 4 : 1024 / D; }
static long join_blocks(int D, int parts, long R) {
  const int rpb = 256 / (D / 4 * join_groups(D, parts));
  return (R + rpb - 1) / rpb;
}
template <int D>
static void join_parts(int parts, hipStream_t st, const PAttnArgs& a) {
  const dim3 grid((unsigned)join_blocks(D, parts, a.R));
  const int groups = join_groups(D, parts);
  if (groups == 1) hipLaunchKernelGGL((prefix_attn_join_kernel<D, 1, 8>), grid, dim3(256), 0, st, a);
  else if (groups == 4) hipLaunchKernelGGL((prefix_attn_join_kernel<D, 4, 4>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((prefix_attn_join_kernel<D, 1024 / D, 4>), grid, dim3(256), 0, st, a);
}

}  // namespace slx

using namespace slx;

extern "C" {

int slx_kv_append(const slx_kv_append_desc* d, slx_stream_t s) {
  SLX_CHECK_ARG(d != nullptr, "slx_kv_append: null desc");
  if (int rc = check_pool(d->pool, "slx_kv_append")) return rc;
  SLX_CHECK_ARG(d->rows >= 0 && d->Hq >= 0 && d->n_seq > 0 && d->cols > 0 && d->ldt >= d->cols,
                "slx_kv_append: rows, Hq >= 0, n_seq > 0, ldt >= cols > 0");
  SLX_CHECK_ARG(d->seq || d->rows_per_seq > 0, "slx_kv_append: seq or rows_per_seq > 0");
  SLX_CHECK_ARG((d->cos_tab == nullptr) == (d->sin_tab == nullptr) && (!d->cos_tab || d->rope_rows > 0),
                "slx_kv_append: cos and sin go together, with rope_rows > 0");
  if (d->rows == 0) return 0;
  SLX_CHECK_ARG(d->qkv && d->table && d->pos, "slx_kv_append: null argument");
  SLX_CHECK_ARG(((uintptr_t)d->qkv & 15) == 0 && d->ldqkv % 8 == 0 && ((uintptr_t)d->q_out & 15) == 0 && d->ldq % 8 == 0,
                "slx_kv_append: qkv and q_out rows must be 16-B aligned");
  SLX_CHECK_ARG(!d->q_out || d->rows == 1 || d->ldq >= (int64_t)d->Hq * d->pool.head_dim, "slx_kv_append: rows of q_out overlap (ldq < Hq * head_dim)");
  SLX_CHECK_ARG((((uintptr_t)d->cos_tab | (uintptr_t)d->sin_tab) & 15) == 0, "slx_kv_append: cos and sin must be 16-B aligned");
  AppendArgs a{view(d->pool), (const bf16*)d->qkv, (long)d->ldqkv, (bf16*)d->q_out, (long)d->ldq, d->table, (long)d->ldt,
               d->n_seq, d->cols, d->seq, d->rows_per_seq > 0 ? d->rows_per_seq : 1, d->pos, (long)d->rows, d->Hq,
               d->pool.heads, d->rope_rows, d->cos_tab, d->sin_tab, 1};
  const long items = (long)((d->q_out ? d->Hq : 0) + 2 * d->pool.heads) * (d->pool.head_dim / 16);
  SLX_CHECK_ARG(items < (1 << 24), "slx_kv_append: too many heads");
  a.rows_per_block = items >= 256 ? 1 : (int)(256 / items);
  const long blocks = (d->rows + a.rows_per_block - 1) / a.rows_per_block;
  SLX_CHECK_ARG(launch_fits(blocks, 256), "slx_kv_append: too many rows");
  if (d->pool.head_dim == 64) hipLaunchKernelGGL(kv_append_kernel<64>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)s, a);
  else hipLaunchKernelGGL(kv_append_kernel<128>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)s, a);
  SLX_LAUNCH_CHECK("slx_kv_append");
  return 0;
}

int64_t slx_prefix_attn_ws_floats(const slx_prefix_attn_desc* d) {
  int capp, capo;
  if (int rc = check_attn(d, &capp, &capo)) return rc;
  const PAttnPlan p = plan_attn(d, capp, capo);
  if (is_direct(p)) return 0;
  return (int64_t)(p.nsp + p.nso) * d->groups * d->width * d->n_q * d->Hq * (d->own_pool.head_dim + 2);
}

int slx_prefix_attn(const slx_prefix_attn_desc* d, slx_stream_t s) {
  int capp, capo;
  if (int rc = check_attn(d, &capp, &capo)) return rc;
  if (d->groups == 0) return 0;
  SLX_CHECK_ARG(d->q && d->out && d->otab && d->olen, "slx_prefix_attn: null argument");
  SLX_CHECK_ARG((((uintptr_t)d->q | (uintptr_t)d->out) & 15) == 0 && d->ldq % 8 == 0 && d->ldo % 8 == 0,
                "slx_prefix_attn: q and out rows must be 16-B aligned");
  const int D = d->own_pool.head_dim, Hkv = d->own_pool.heads;
  SLX_CHECK_ARG(d->ldo >= (int64_t)d->Hq * D || (int64_t)d->groups * d->width * d->n_q == 1, "slx_prefix_attn: rows of out overlap (ldo < Hq * head_dim)");
  const PAttnPlan p = plan_attn(d, capp, capo);
  PAttnArgs a;
  memset(&a, 0, sizeof(a));
  a.q = (const bf16*)d->q; a.ldq = d->ldq; a.out = (bf16*)d->out; a.ldo = d->ldo; a.lse = d->lse;
  a.own = Seg{view(d->own_pool), d->otab, (long)d->ldot, d->olen, capo, p.nso};
  if (p.nsp > 0) a.pre = Seg{view(d->prefix_pool), d->ptab, (long)d->ldpt, d->plen, capp, p.nsp};
  a.W = d->width; a.Tq = d->n_q; a.Hq = d->Hq; a.Hkv = Hkv; a.gq = d->Hq / Hkv;
  a.c = d->scale * 1.44269504088896341f;
  a.gmul = a.gq == 1 ? 0u : (unsigned)((1ull << 32) / a.gq + 1);
  a.mt_pre = p.mtp; a.mt_own = p.mto; a.groups = d->groups;
  const long n_pre = p.whole ? 0 : ((long)d->groups * Hkv * p.nsp + 7) / 8 * 8 * p.mtp;
  a.D = D;
  a.direct = is_direct(p);
  a.R = (long)d->groups * d->width * d->n_q * d->Hq;
  a.ws = d->ws;
  const int64_t need = a.direct ? 0 : (int64_t)(p.nsp + p.nso) * a.R * (D + 2);
  SLX_CHECK_ARG(need == 0 || (d->ws && ((uintptr_t)d->ws & 15) == 0 && d->ws_floats >= need),
                "slx_prefix_attn: needs a 16-B aligned workspace of %lld floats", (long long)need);
  const long blocks = n_pre + (long)d->groups * d->width * Hkv * p.mto * p.nso;
  SLX_CHECK_ARG(launch_fits(blocks, p.whole ? 64 * p.whole : 256) && (a.direct || launch_fits(join_blocks(D, p.nsp + p.nso, a.R), 256)),
                "slx_prefix_attn: too many rows");
  a.n_pre = (unsigned)n_pre;
  const bool known = D == 64 ? launch_attn<64>(p, dim3((unsigned)blocks), (hipStream_t)s, a)
                             : launch_attn<128>(p, dim3((unsigned)blocks), (hipStream_t)s, a);
  SLX_CHECK_ARG(known, "slx_prefix_attn: no kernel for row tiles %d and %d", p.kp, p.ko);
  SLX_LAUNCH_CHECK("slx_prefix_attn");
  if (!a.direct) {
    if (D == 64) join_parts<64>(p.nsp + p.nso, (hipStream_t)s, a);
    else join_parts<128>(p.nsp + p.nso, (hipStream_t)s, a);
    SLX_LAUNCH_CHECK("slx_prefix_attn (join)");
  }
  return 0;
}

}  // extern "C"
