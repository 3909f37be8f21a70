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
// One thread takes the pair of 8-element chunks c and c + D/16 of one head (16-B loads and stores).
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
// The prefix of a group is read once for all of its width * n_q * (Hq / Hkv) query rows of a kv head: a workgroup
// takes 16 * NQ of those rows and one range of the prefix, whose 32-key tiles its 4 waves share out; the sequences'
// own keys are workgroups of the same launch, with the n_q * (Hq / Hkv) rows of one sequence. Each writes (m, l, o) of
// its range, and a second launch joins a row's parts.
//
// Per tile and wave: S^T = K Q^T on v_mfma_f32_16x16x32_bf16 with the keys as rows and the queries as columns, so a
// lane holds 8 keys of ONE query, and the probabilities are already the B operand of O^T += V^T P^T (the sum over keys
// may take them in any order: slot j of lane group q is key 4q + j, or 16 + 4q + j - 4). V^T's A operand needs 8 keys
// of one d: a lane loads D/16 neighbouring d of each of its 8 keys and pairs them with v_perm_b32 (the MFMA row r of
// product e stands for d = (D/16) r + e), so nothing goes through LDS before the final merge of the waves.
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
  float c;  // scale * log2(e)
  int mt_pre, mt_own;
  long n_pre;  // workgroups of the prefix part
  int direct;  // one part per row: the workgroups write the output themselves
  long R;      // rows * Hq
  float* ws;   // o [parts][R][D], then (m, l) [parts][R]
};

__host__ __device__ __forceinline__ int split_keys(int len, int ns) { return ((len + ns - 1) / ns + 127) & ~127; }
__device__ __forceinline__ int seg_len(const Seg& s, long i) { return s.len ? max(0, min(s.len[i], s.cap)) : 0; }

template <int D, int NQ>
__device__ __forceinline__ void attn_item(const PAttnArgs& a, const Seg& sg, const int* tab, bool causal, int len, int kb,
                                          int ke, int kvh, long tok0, int ntok, int mt, int part, char* smem) {
  constexpr int KK = D / 32, NE = D / 16;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, grp = lane >> 4;
  const int rows = ntok * a.gq, r0 = mt * 16 * NQ;
  const int shift = sg.p.shift, mask = (1 << shift) - 1;
  const unsigned npg = (unsigned)sg.p.n_pages;
  const bf16* kbase = sg.p.k + kvh * sg.p.hs + 8 * grp;
  const bf16* vbase = sg.p.v + kvh * sg.p.hs + NE * col;
  // the causal edge of an own segment: token t of Tq sees keys <= len - Tq + t
  const int tmin = r0 / a.gq, tmax = (min(r0 + 16 * NQ, rows) - 1) / a.gq;
  const int free_end = causal ? min(ke, len - a.Tq + tmin + 1) : ke;  // keys below it are seen by every row
  if (causal) ke = min(ke, len - a.Tq + tmax + 1);

  bf16x8 qf[NQ][KK];
  int lim[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int r = min(r0 + 16 * n + col, rows - 1), t = r / a.gq;
    const bf16* qp = a.q + (tok0 + t) * a.ldq + (long)(kvh * a.gq + r - t * a.gq) * D + 8 * grp;
#pragma unroll
    for (int k = 0; k < KK; ++k) qf[n][k] = *reinterpret_cast<const bf16x8*>(qp + 32 * k);
    lim[n] = causal ? min(ke, len - a.Tq + t + 1) : ke;
  }

  float m[NQ], l[NQ];
  f32x4 o[NQ][NE];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    m[n] = -INFINITY;
    l[n] = 0.f;
#pragma unroll
    for (int e = 0; e < NE; ++e) o[n][e] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  bf16x8 kf[2][KK];
  unsigned vr[8][NE / 2];  // NE d of each of the lane's 8 keys
  bool vok[8];
  const bool fine = shift < 2;  // pages of 1 or 2 slots: a page number for each key of a lane's four
  auto entry = [&](int key) { return tab[min(key, len - 1) >> shift]; };
  auto offset = [&](int e, int key) {
    return (unsigned)e < npg ? (long)e * sg.p.ps + (long)(min(key, len - 1) & mask) * sg.p.ss : 0L;
  };
  int ek[2], ev[2];  // page numbers of the next tile to load
  auto entries_k = [&](int k0) {
    if (k0 >= ke) return;
#pragma unroll
    for (int s = 0; s < 2; ++s) ek[s] = entry(k0 + 16 * s + col);
  };
  auto entries_v = [&](int k0) {
    if (k0 >= ke || fine) return;
#pragma unroll
    for (int s = 0; s < 2; ++s) ev[s] = entry(k0 + 16 * s + 4 * grp);
  };
  auto load_k = [&](int k0) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const bf16* p = kbase + offset(ek[s], k0 + 16 * s + col);
#pragma unroll
      for (int k = 0; k < KK; ++k) kf[s][k] = *reinterpret_cast<const bf16x8*>(p + 32 * k);
    }
  };
  auto load_v = [&](int k0) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int key = k0 + 16 * (j >> 2) + 4 * grp + (j & 3);
      const int e = fine ? entry(key) : ev[j >> 2];
      vok[j] = (unsigned)e < npg && key < len;
      const bf16* p = vbase + offset(e, key);
      if constexpr (NE == 4) {
        const u32x2 x = *reinterpret_cast<const u32x2*>(p);
        vr[j][0] = x[0]; vr[j][1] = x[1];
      } else {
        const u32x4 x = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
        for (int i = 0; i < NE / 2; ++i) vr[j][i] = x[i];
      }
    }
  };

  int k0 = kb + 32 * wave;
  if (k0 < ke) {
    entries_k(k0);
    entries_v(k0);
    load_k(k0);
    load_v(k0);
    entries_k(k0 + 128);
    entries_v(k0 + 128);
  }
  for (; k0 < ke; k0 += 128) {
    f32x4 s[NQ][2];
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s[n][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KK; ++k) s[n][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[h][k], qf[n][k], s[n][h], 0, 0, 0);
      }
    bool good = true;
#pragma unroll
    for (int j = 0; j < 8; ++j) good = good && vok[j];
    const bool edge = k0 + 32 > free_end || __any(!good);
    bool vk[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) vk[j] = vok[j];
    if (k0 + 128 < ke) {
      load_k(k0 + 128);
      entries_k(k0 + 256);
    }
    bf16x8 pb[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = s[n][j >> 2][j & 3] * a.c;
      if (edge) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!vk[j] || k0 + 16 * (j >> 2) + 4 * grp + (j & 3) >= lim[n]) x[j] = -INFINITY;
      }
      float mx = x[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) mx = fmaxf(mx, x[j]);
      // the running maximum moves only when a score passes it by 2^8 (exact all the same: it cancels in o / l)
      if (__any(mx > m[n] + 8.0f)) {
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float mn = fmaxf(m[n], mx);
        const float r = m[n] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[n] - mn);
        m[n] = mn;
        l[n] *= r;
#pragma unroll
        for (int e = 0; e < NE; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[n][e][i] *= r;
      }
      const float mu = m[n] == -INFINITY ? 0.f : m[n];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        // P in bf16 for the MFMA (half a step, 2^-9 of each term, as the output itself is rounded); l sums the same
        // rounded values, so what is left is the terms' own scatter
        const float p = __builtin_amdgcn_exp2f(x[j] - mu);
        pb[n][j] = (bf16)p;
        l[n] += (float)pb[n][j];
      }
    }
    if (edge) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < NE / 2; ++i) vr[j][i] = vk[j] ? vr[j][i] : 0u;
      if (causal && k0 + 32 > free_end) {
        // keys that some row does not see yet: 0 * inf would reach it through the MFMA, so non-finite values leave the
        // operand and are added to the rows that see them
        bool odd = false;
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int i = 0; i < NE / 2; ++i) {
            const unsigned x = vr[j][i];
            const bool lo = (x & 0x7F80u) == 0x7F80u, hi = (x & 0x7F800000u) == 0x7F800000u;
            odd = odd || lo || hi;
            vr[j][i] = (lo ? 0u : (x & 0xFFFFu)) | (hi ? 0u : (x & 0xFFFF0000u));
          }
        if (__any(odd)) {
          for (int kk = 0; kk < 32 && k0 + kk < ke; ++kk) {
            const int e = entry(k0 + kk);
            if ((unsigned)e >= npg) continue;
            const bf16* p = sg.p.v + kvh * sg.p.hs + offset(e, k0 + kk) + (D / 4) * grp;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int ee = 0; ee < NE; ++ee) {
                const float v = (float)p[NE * i + ee];
                const bool nf = !(fabsf(v) < INFINITY);
#pragma unroll
                for (int n = 0; n < NQ; ++n)
                  if (nf && k0 + kk < lim[n]) o[n][ee][i] += v;
              }
          }
        }
      }
    }
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      union { unsigned u[4]; bf16x8 b; } vt;
#pragma unroll
      for (int p = 0; p < 4; ++p)
        vt.u[p] = __builtin_amdgcn_perm(vr[2 * p + 1][e >> 1], vr[2 * p][e >> 1], (e & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
      for (int n = 0; n < NQ; ++n) o[n][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt.b, pb[n], o[n][e], 0, 0, 0);
    }
    if (k0 + 128 < ke) {
      load_v(k0 + 128);
      entries_v(k0 + 256);
    }
  }

  // ---- the 4 waves' (m, l, o) into one: waves 2, 3 hand theirs to 0, 1, then 1 to 0
  float* sm = reinterpret_cast<float*>(smem);      // [4][16 NQ]
  float* sl = sm + 4 * 16 * NQ;                    // [4][16 NQ]
  f32x4* so = reinterpret_cast<f32x4*>(sl + 4 * 16 * NQ);  // [2][NQ * NE][64 lanes]
  float M[NQ], L[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    l[n] += __shfl_xor(l[n], 16, 64);
    l[n] += __shfl_xor(l[n], 32, 64);
    if (grp == 0) {
      sm[wave * 16 * NQ + 16 * n + col] = m[n];
      sl[wave * 16 * NQ + 16 * n + col] = l[n];
    }
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    float mw[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) mw[w] = sm[w * 16 * NQ + 16 * n + col];
    M[n] = fmaxf(fmaxf(mw[0], mw[1]), fmaxf(mw[2], mw[3]));
    L[n] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w)
      L[n] += mw[w] == -INFINITY ? 0.f : sl[w * 16 * NQ + 16 * n + col] * __builtin_amdgcn_exp2f(mw[w] - M[n]);
    const float r = m[n] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[n] - M[n]);
#pragma unroll
    for (int e = 0; e < NE; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][e][i] *= r;
  }
  if (wave >= 2) {
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int e = 0; e < NE; ++e) so[((wave - 2) * NQ * NE + n * NE + e) * 64 + lane] = o[n][e];
  }
  __syncthreads();
  if (wave < 2) {
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int e = 0; e < NE; ++e) o[n][e] += so[(wave * NQ * NE + n * NE + e) * 64 + lane];
  }
  __syncthreads();
  if (wave == 1) {
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int e = 0; e < NE; ++e) so[(n * NE + e) * 64 + lane] = o[n][e];
  }
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int r = r0 + 16 * n + col;
    if (r >= rows) continue;
    const int t = r / a.gq, head = kvh * a.gq + r - t * a.gq;
    const long row = (tok0 + t) * a.Hq + head;
    float x[4 * NE];  // d = (D/4) grp + NE i + e
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      o[n][e] += so[(n * NE + e) * 64 + lane];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[NE * i + e] = o[n][e][i];
    }
    if (a.direct) {
      const float inv = L[n] > 0.f || L[n] != L[n] ? 1.0f / L[n] : 0.f;  // no key seen: zeros
      bf16* op = a.out + (tok0 + t) * a.ldo + (long)head * D + (D / 4) * grp;
#pragma unroll
      for (int b = 0; b < NE / 2; ++b) {
        bf16x8 y;
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = (bf16)(x[8 * b + j] * inv);
        *reinterpret_cast<bf16x8*>(op + 8 * b) = y;
      }
      if (a.lse && grp == 0) a.lse[row] = M[n] == -INFINITY ? -INFINITY : (M[n] + log2f(L[n])) * 0.69314718055994531f;
    } else {
      float* op = a.ws + ((long)part * a.R + row) * D + (D / 4) * grp;
#pragma unroll
      for (int b = 0; b < NE; ++b) *reinterpret_cast<f32x4*>(op + 4 * b) = f32x4{x[4 * b], x[4 * b + 1], x[4 * b + 2], x[4 * b + 3]};
      if (grp == 0) {
        float* ml = a.ws + (long)(a.pre.ns + a.own.ns) * a.R * D + ((long)part * a.R + row) * 2;
        *reinterpret_cast<float2*>(ml) = make_float2(M[n], L[n]);
      }
    }
  }
}

template <int D, int NQP, int NQO>
__global__ __launch_bounds__(256, 2) void prefix_attn_kernel(PAttnArgs a) {
  constexpr int NQ = NQP > NQO ? NQP : NQO;
  __shared__ __attribute__((aligned(16))) char smem[2 * 4 * 16 * NQ * 4 + 2 * NQ * (D / 16) * 64 * 16];
  long b = blockIdx.x;
  if (b < a.n_pre) {  // [row tile][group][kv head][range]
    const int sp = (int)(b % a.pre.ns);
    b /= a.pre.ns;
    const int kvh = (int)(b % a.Hkv);
    b /= a.Hkv;
    const long ng = a.n_pre / ((long)a.pre.ns * a.Hkv * a.mt_pre);
    const long g = b % ng;
    const int mt = (int)(b / ng);
    const int len = seg_len(a.pre, g), ks = split_keys(len, a.pre.ns), kb = sp * ks;
    if (kb >= len) return;
    attn_item<D, NQP>(a, a.pre, a.pre.tab + g * a.pre.ldt, false, len, kb, min(len, kb + ks), kvh, g * a.W * a.Tq,
                      a.W * a.Tq, mt, sp, smem);
  } else {  // [sequence][row tile][kv head][range]
    b -= a.n_pre;
    const int sp = (int)(b % a.own.ns);
    b /= a.own.ns;
    const int kvh = (int)(b % a.Hkv);
    b /= a.Hkv;
    const int mt = (int)(b % a.mt_own);
    const long n = b / a.mt_own;
    const int len = seg_len(a.own, n), ks = split_keys(len, a.own.ns), kb = sp * ks;
    if (kb >= len && !(a.direct && sp == 0)) return;
    attn_item<D, NQO>(a, a.own, a.own.tab + n * a.own.ldt, true, len, kb, min(len, kb + ks), kvh, n * a.Tq, a.Tq, mt,
                      a.pre.ns + sp, smem);
  }
}

// joins the parts of a row: D / 4 threads a row, four d a thread
template <int D>
__global__ __launch_bounds__(256) void prefix_attn_join_kernel(PAttnArgs a) {
  constexpr int TPR = D / 4;
  const long row = ((long)blockIdx.x * 256 + threadIdx.x) / TPR;
  const int d = (threadIdx.x % TPR) * 4;
  if (row >= a.R) return;
  const long tok = row / a.Hq, n = tok / a.Tq;
  const int pl = seg_len(a.pre, n / a.W), ol = seg_len(a.own, n);
  const int np = pl ? (pl + split_keys(pl, a.pre.ns) - 1) / split_keys(pl, a.pre.ns) : 0;
  const int no = ol ? (ol + split_keys(ol, a.own.ns) - 1) / split_keys(ol, a.own.ns) : 0;
  const float2* ml = reinterpret_cast<const float2*>(a.ws + (long)(a.pre.ns + a.own.ns) * a.R * D) + row;
  const float* ob = a.ws + row * D + d;
  float m = -INFINITY, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  constexpr int B = 4;
  for (int i0 = 0; i0 < np + no; i0 += B) {
    float2 x[B];
    f32x4 y[B];
#pragma unroll
    for (int u = 0; u < B; ++u) {
      const int i = min(i0 + u, np + no - 1), p = i < np ? i : a.pre.ns + i - np;
      x[u] = ml[(long)p * a.R];
      y[u] = *reinterpret_cast<const f32x4*>(ob + (long)p * a.R * D);
      if (i0 + u >= np + no) x[u].x = -INFINITY;
    }
    float mn = m;
#pragma unroll
    for (int u = 0; u < B; ++u) mn = fmaxf(mn, x[u].x);
    const float r = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
    l *= r;
    o *= r;
#pragma unroll
    for (int u = 0; u < B; ++u) {
      if (x[u].x == -INFINITY) continue;  // its o was not computed from any key
      const float w = __builtin_amdgcn_exp2f(x[u].x - mn);
      l = __builtin_fmaf(w, x[u].y, l);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = __builtin_fmaf(w, y[u][j], o[j]);
    }
    m = mn;
  }
  const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
  bf16x4 y;
#pragma unroll
  for (int j = 0; j < 4; ++j) y[j] = (bf16)(o[j] * inv);
  *reinterpret_cast<bf16x4*>(a.out + tok * a.ldo + (row - tok * a.Hq) * D + d) = y;
  if (a.lse && d == 0) a.lse[row] = m == -INFINITY ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
}

// Row tiles and key ranges of a call: a rule on sizes and the host's bounds alone, so a captured call replays for any
// lengths up to them. 16, 32 or (head size 64) 64 rows a workgroup, the fewest that hold all rows that share the keys;
// as many ranges as give about kTarget workgroups, each of at least 128 keys (one tile a wave).
constexpr long kTarget = 1024;
struct PAttnPlan { int nqp, nqo, mtp, mto, nsp, nso; };
static PAttnPlan plan_attn(const slx_prefix_attn_desc* d, int capp, int capo) {
  PAttnPlan p;
  const int gq = d->Hq / d->own_pool.heads, most = d->own_pool.head_dim == 64 ? 4 : 2;
  auto tile = [&](long rows) { return rows <= 16 ? 1 : (rows <= 32 || most == 2) ? 2 : 4; };
  const long rp = (long)d->width * d->n_q * gq, ro = (long)d->n_q * gq;
  p.nqo = tile(ro);
  p.nqp = capp > 0 ? tile(rp) : p.nqo;
  p.mtp = (int)((rp + 16 * p.nqp - 1) / (16 * p.nqp));
  p.mto = (int)((ro + 16 * p.nqo - 1) / (16 * p.nqo));
  const long up = (capp + 127) / 128, uo = (capo + 127) / 128;  // units of 128 keys
  const long ip = (long)d->groups * d->own_pool.heads * p.mtp, io = (long)d->groups * d->width * d->own_pool.heads * p.mto;
  const long per = (ip * up + io * uo + kTarget - 1) / kTarget, u = per > 1 ? per : 1;
  p.nsp = (int)((up + u - 1) / u);
  p.nso = (int)((uo + u - 1) / u);
  if (p.nso < 1) p.nso = 1;
  return p;
}

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
  return 0;
}

template <int D>
static void launch_attn(const PAttnPlan& p, dim3 grid, hipStream_t st, const PAttnArgs& a) {
#define SLX_PA(P, O)                                                                                         \
  if (p.nqp == P && p.nqo == O) {                                                                            \
    hipLaunchKernelGGL((prefix_attn_kernel<D, P, O>), grid, dim3(256), 0, st, a);                            \
    return;                                                                                                  \
  }
  SLX_PA(1, 1) SLX_PA(2, 1) SLX_PA(2, 2)
  if constexpr (D == 64) { SLX_PA(4, 1) SLX_PA(4, 2) SLX_PA(4, 4) }
#undef SLX_PA
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
  SLX_CHECK_ARG((((uintptr_t)d->cos_tab | (uintptr_t)d->sin_tab) & 15) == 0, "slx_kv_append: cos and sin must be 16-B aligned");
  AppendArgs a{view(d->pool), (const bf16*)d->qkv, (long)d->ldqkv, (bf16*)d->q_out, (long)d->ldq, d->table, (long)d->ldt,
               d->n_seq, d->cols, d->seq, d->rows_per_seq > 0 ? d->rows_per_seq : 1, d->pos, (long)d->rows, d->Hq,
               d->pool.heads, d->rope_rows, d->cos_tab, d->sin_tab, 1};
  const long items = (long)((d->q_out ? d->Hq : 0) + 2 * d->pool.heads) * (d->pool.head_dim / 16);
  SLX_CHECK_ARG(items < (1 << 24), "slx_kv_append: too many heads");
  a.rows_per_block = items >= 256 ? 1 : (int)(256 / items);
  const long blocks = (d->rows + a.rows_per_block - 1) / a.rows_per_block;
  SLX_CHECK_ARG(blocks < 2147483648L, "slx_kv_append: too many rows");
  if (d->pool.head_dim == 64) hipLaunchKernelGGL(kv_append_kernel<64>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)s, a);
  else hipLaunchKernelGGL(kv_append_kernel<128>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)s, a);
  SLX_LAUNCH_CHECK("slx_kv_append");
  return 0;
}

int64_t slx_prefix_attn_ws_floats(const slx_prefix_attn_desc* d) {
  int capp, capo;
  if (int rc = check_attn(d, &capp, &capo)) return rc;
  const PAttnPlan p = plan_attn(d, capp, capo);
  if (p.nsp + p.nso == 1) return 0;
  return (int64_t)(p.nsp + p.nso) * d->groups * d->width * d->n_q * d->Hq * (d->own_pool.head_dim + 2);
}

int slx_prefix_attn(const slx_prefix_attn_desc* d, slx_stream_t s) {
  int capp, capo;
  if (int rc = check_attn(d, &capp, &capo)) return rc;
  if (d->groups == 0) return 0;
  SLX_CHECK_ARG(d->q && d->out && d->otab && d->olen, "slx_prefix_attn: null argument");
  SLX_CHECK_ARG((((uintptr_t)d->q | (uintptr_t)d->out) & 15) == 0 && d->ldq % 8 == 0 && d->ldo % 8 == 0,
                "slx_prefix_attn: q and out rows must be 16-B aligned");
  const PAttnPlan p = plan_attn(d, capp, capo);
  const int D = d->own_pool.head_dim, Hkv = d->own_pool.heads;
  PAttnArgs a;
  memset(&a, 0, sizeof(a));
  a.q = (const bf16*)d->q; a.ldq = d->ldq; a.out = (bf16*)d->out; a.ldo = d->ldo; a.lse = d->lse;
  a.own = Seg{view(d->own_pool), d->otab, (long)d->ldot, d->olen, capo, p.nso};
  if (p.nsp > 0) a.pre = Seg{view(d->prefix_pool), d->ptab, (long)d->ldpt, d->plen, capp, p.nsp};
  a.W = d->width; a.Tq = d->n_q; a.Hq = d->Hq; a.Hkv = Hkv; a.gq = d->Hq / Hkv;
  a.c = d->scale * 1.44269504088896341f;
  a.mt_pre = p.mtp; a.mt_own = p.mto;
  a.n_pre = (long)d->groups * Hkv * p.mtp * p.nsp;
  a.direct = p.nsp + p.nso == 1;
  a.R = (long)d->groups * d->width * d->n_q * d->Hq;
  a.ws = d->ws;
  const int64_t need = a.direct ? 0 : (int64_t)(p.nsp + p.nso) * a.R * (D + 2);
  SLX_CHECK_ARG(need == 0 || (d->ws && ((uintptr_t)d->ws & 15) == 0 && d->ws_floats >= need),
                "slx_prefix_attn: needs a 16-B aligned workspace of %lld floats", (long long)need);
  const long blocks = a.n_pre + (long)d->groups * d->width * Hkv * p.mto * p.nso;
  SLX_CHECK_ARG(blocks < 2147483648L, "slx_prefix_attn: too many rows");
  if (D == 64) launch_attn<64>(p, dim3((unsigned)blocks), (hipStream_t)s, a);
  else launch_attn<128>(p, dim3((unsigned)blocks), (hipStream_t)s, a);
  SLX_LAUNCH_CHECK("slx_prefix_attn");
  if (!a.direct) {
    const long jb = (a.R * (D / 4) + 255) / 256;
    if (D == 64) hipLaunchKernelGGL(prefix_attn_join_kernel<64>, dim3((unsigned)jb), dim3(256), 0, (hipStream_t)s, a);
    else hipLaunchKernelGGL(prefix_attn_join_kernel<128>, dim3((unsigned)jb), dim3(256), 0, (hipStream_t)s, a);
    SLX_LAUNCH_CHECK("slx_prefix_attn (join)");
  }
  return 0;
}

}  // extern "C"
