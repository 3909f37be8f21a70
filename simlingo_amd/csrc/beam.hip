// Beam search on the device: the choice of the k best continuations over all beams and the whole vocabulary, and the
// reordering of any state by the beams chosen. They stand beside the greedy choice (simlingo_training/models/
// language_model/llm.py:145-160 argmax; decode.hip folds it into the LM head).
//
// score(b, w, t) = s[b, w] + x[b, w, t] - log sum_t' e^{x[b, w, t']}; the k largest of a batch entry's width * V
// scores, ties to the lowest w * V + t. One pass over the logits: within a row the order of the scores is the order of
// the logits, so every 4096-column chunk hands on its k largest logits and its (max, sum) of the softmax, and the
// second launch forms the row sums, the scores (64 bits, from exact 32-bit maxima and sums of at most 4096 terms each)
// and the k best of all rows.
//
// Measured: 4 rows of 151655 f32 logits, 4 chosen: 4.8 + 4.8 us (the logits alone: 0.5 us at 5.2 TB/s); 8 x 8 rows of bf16, a
// quarter of them at their end, 16 chosen: 10.6 + 7.4 us (2.8). Bound by latency (a launch takes 2 us, the chain load -> maximum
// -> threshold -> candidates -> rank with two barriers 3) and, where seven workgroups share a CU, by the instructions of that
// chain; the second launch has one workgroup a batch entry, a wave a row: scores, lists, logarithm, ranks, the last ranking.
// 8192 columns a workgroup instead: 2 us more, at 8 x 16 rows of f32, 32 chosen, 3 of 37.
#include <type_traits>

#include "common.h"
#include "../../include/slx.h"

namespace slx {

typedef unsigned long long u64;
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
constexpr int kSelChunk = 4096;          // columns a workgroup: 16 a thread
constexpr int kSelMaxChunks = 64;        // one lane each in the second launch
constexpr int kSelMaxK = 64, kSelMaxW = 64;
constexpr int kSelList = 256;            // candidates of a chunk (64 a wave), or of a row's lists, that are ranked at once
constexpr int kSelFew = 512;             // entries of the rows' lists that are ranked at once: 16 x 32 in 20.4 us, k rounds of the largest head 27.7

struct SelArgs {
  const void* x; long ldx;
  const float* score; const unsigned char* fin;
  float* score_out; int *parent, *token; unsigned char* fin_out;
  int B, W, V, K, C, pad, eos;  // C: chunks a row
  float2* ml;  // [B * W][C] (max, sum)
  u64* keys;   // [B * W][C][K], descending; 0 = none
};

// order-preserving bits of a float; NaN below everything (its row's sum is NaN, so the row offers nothing)
__device__ __forceinline__ unsigned ord_f(float v) {
  const unsigned u = __float_as_uint(v);
  return v != v ? 0u : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float unord_f(unsigned u) {
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7FFFFFFFu) : ~u);
}
__device__ __forceinline__ u64 key_of(unsigned ord, int idx) { return ((u64)ord << 32) | (0xFFFFFFFFu - (unsigned)idx); }
__device__ __forceinline__ int key_idx(u64 k) { return (int)(0xFFFFFFFFu - (unsigned)k); }

// the largest of a value over the wave: DPP within rows of 16 lanes, then the 4 rows' results
template <int CTRL>
__device__ __forceinline__ unsigned dpp_u(unsigned v) {
  return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}
__device__ __forceinline__ unsigned wave_umax(unsigned x) {
  x = max(x, dpp_u<0xB1>(x));   // quad_perm [1,0,3,2]
  x = max(x, dpp_u<0x4E>(x));   // quad_perm [2,3,0,1]
  x = max(x, dpp_u<0x141>(x));  // row_half_mirror
  x = max(x, dpp_u<0x140>(x));  // row_mirror
  const unsigned a = (unsigned)__builtin_amdgcn_readlane((int)x, 0), b = (unsigned)__builtin_amdgcn_readlane((int)x, 16);
  const unsigned c = (unsigned)__builtin_amdgcn_readlane((int)x, 32), d = (unsigned)__builtin_amdgcn_readlane((int)x, 48);
  return max(max(a, b), max(c, d));
}
__device__ __forceinline__ float wave_fsum(float x) {
  x += __uint_as_float(dpp_u<0xB1>(__float_as_uint(x)));
  x += __uint_as_float(dpp_u<0x4E>(__float_as_uint(x)));
  x += __uint_as_float(dpp_u<0x141>(__float_as_uint(x)));
  x += __uint_as_float(dpp_u<0x140>(__float_as_uint(x)));
  const auto rl = [&](int l) { return __uint_as_float((unsigned)__builtin_amdgcn_readlane(__float_as_int(x), l)); };
  return (rl(0) + rl(16)) + (rl(32) + rl(48));
}
// the largest key over the wave (uniform): high words first, then the low words of the lanes that hold that high word
__device__ __forceinline__ u64 wave_kmax(u64 k) {
  const unsigned hi = wave_umax((unsigned)(k >> 32));
  const unsigned lo = wave_umax((unsigned)(k >> 32) == hi ? (unsigned)k : 0u);
  return ((u64)hi << 32) | lo;
}

// what one lane of a wave has put into LDS is there for the others (its accesses are in order; the compiler keeps them so)
__device__ __forceinline__ void wave_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// A value with at least K of the wave's N x 64 values at or above it, given that lo has: halved into between lo and the largest
// until few more than K are left (all of 20 halvings leave a range of 2^12 of a float's bits; more than K is only more work).
template <int N>
__device__ __forceinline__ unsigned kth_below(const unsigned (&x)[N], unsigned lo, unsigned hi, int K) {
  auto above = [&](unsigned t) {
    int k = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) k += __popcll(__ballot(x[i] >= t));
    return k;
  };
  const unsigned near = hi - min(hi - lo, 0x02000000u);  // most often within a factor of 16 of the largest
  if (near > lo && above(near) >= K) lo = near;
  for (int it = 0; it < 20 && lo < hi; ++it) {
    const unsigned mid = lo + (hi - lo) / 2 + 1;
    const int k = above(mid);
    if (k >= K) lo = mid;
    else hi = mid - 1;
    if (k >= K && k <= K + 2) break;
  }
  return lo;
}

template <typename T>
__global__ __launch_bounds__(256) void beam_chunk_kernel(SelArgs a) {
  __shared__ float2 sml[4];
  __shared__ unsigned smax[256];
  __shared__ int scount[4];
  __shared__ u64 list[kSelList];  // 64 a wave
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = (int)(blockIdx.x / (unsigned)a.C), c = (int)(blockIdx.x - (unsigned)row * a.C);
  constexpr int E = kSelChunk / 256, VEC = 16 / (int)sizeof(T), U = E / VEC, CHUNK = kSelChunk;  // 16-B loads, VEC columns each
  const T* xr = (const T*)a.x + (long)row * a.ldx;
  const int c0 = c * CHUNK;
  // the last chunk is read element by element and spread over all threads; a thread's columns rise with e, so those below V
  // come first in its order: n of them
  const bool full = c0 + CHUNK <= a.V;
  auto col = [&](int e) { return c0 + (full ? ((e / VEC) * 256 + tid) * VEC + e % VEC : e * 256 + tid); };
  float v[E];
  int n = E;
  // rows that have ended, or are out of the search already, are not read
  const unsigned char ended = a.fin ? a.fin[row] : 0;  // both on their way before either is looked at
  const float s = a.score[row];
  if (ended || !(fabsf(s) < INFINITY)) return;
  if (full) {
    T t[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) __builtin_memcpy(t[u], xr + c0 + (u * 256 + tid) * VEC, 16);  // rows of odd length: any alignment of T
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = (float)t[e / VEC][e % VEC];
  } else {
    n = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool in = col(e) < a.V;
      v[e] = in ? (float)xr[col(e)] : -INFINITY;
      n += in;
    }
  }
  float m = v[0];  // NaN stays out of the maximum, and makes the row's sum NaN, so that the row offers nothing
#pragma unroll
  for (int e = 1; e < E; ++e) m = fmaxf(m, v[e]);
  const unsigned om = ord_f(m);
  const float mw = unord_f(wave_umax(om));
  const float ms = mw == -INFINITY ? 0.f : mw;
  float l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) l += __expf(v[e] - ms);
  l = wave_fsum(l);

  // a threshold with at least K of the chunk's columns at or above it: the K-th largest of the threads' own maxima, halved
  // into from both ends until few more than K are left (-inf: fewer threads than K, or -inf itself)
  smax[tid] = n ? om : 0u;
  if (lane == 0) sml[wave] = make_float2(mw, l);
  if (n < E) {  // columns behind V: above no threshold
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = e < n ? v[e] : NAN;
  }
  __syncthreads();
  float tv = -INFINITY;
  {
    unsigned x[4], mx = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = smax[64 * i + lane];
      mx = max(mx, x[i]);
    }
    if (a.K <= 32) {  // of 64 groups of four threads: a few candidates more, a quarter of the work (12.5 -> 10.5 us of 16 chosen)
      const unsigned y[1] = {mx};
      if (__popcll(__ballot(mx > 0x007FFFFFu)) >= a.K) tv = unord_f(kth_below(y, 0x00800000u, wave_umax(mx), a.K));  // above -inf
    } else {
      int finite = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) finite += __popcll(__ballot(x[i] > 0x007FFFFFu));
      if (finite >= a.K) tv = unord_f(kth_below(x, 0x00800000u, wave_umax(mx), a.K));
    }
  }
  int at = 0;  // this wave's candidates
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const bool h = v[e] >= tv;
    const u64 in = __ballot(h);
    if (in) {
      const int i = at + __popcll(in & ((1ull << lane) - 1));
      if (h && i < 64) list[64 * wave + i] = key_of(ord_f(v[e] + 0.f), col(e));  // -0 ties with 0
      at += __popcll(in);
    }
  }
  if (lane == 0) scount[wave] = at;
  __syncthreads();
  int cnt[4];
  bool over = false;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    cnt[w] = scount[w];
    over = over || cnt[w] > 64;
  }
  if (over) {  // many equal logits: each wave draws its K largest keys one by one
    u64 last = ~0ull;
    for (int i = 0; i < a.K; ++i) {
      u64 best = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const u64 k = key_of(ord_f(v[e] + 0.f), col(e));
        if (v[e] == v[e] && k < last && k > best) best = k;
      }
      best = wave_kmax(best);
      if (lane == 0) list[64 * wave + i] = best;
      last = best;  // 0 once the wave has no more: nothing is below it
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) cnt[w] = a.K;
    __syncthreads();
  }
  u64* out = a.keys + ((long)row * a.C + c) * a.K;
  const int mine = wave == 0 ? cnt[0] : wave == 1 ? cnt[1] : wave == 2 ? cnt[2] : cnt[3];
  if (lane < mine) {  // every key is its own: the rank is the number of greater ones
    const u64 k = list[tid];
    int rank = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll 4
      for (int i = 0; i < cnt[w]; ++i) rank += list[64 * w + i] > k;
    if (k && rank < a.K) out[rank] = k;
  }
  // fewer columns than K (the last chunk): the rest of the list is empty
  const int have = min(a.V - c0, CHUNK);
  if (tid >= have && tid < a.K) out[tid] = 0;
  if (tid == 0) {
    float M = sml[0].x;
    for (int w = 1; w < 4; ++w) M = fmaxf(M, sml[w].x);
    float L = 0.f;
    for (int w = 0; w < 4; ++w) L += sml[w].x == -INFINITY && sml[w].y == 0.f ? 0.f : sml[w].y * __expf(sml[w].x - (M == -INFINITY ? 0.f : M));
    a.ml[(long)row * a.C + c] = make_float2(M, L);
  }
}

__device__ __forceinline__ u64 lane_u64(u64 v, int lane) {
  return ((u64)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32) | (unsigned)__builtin_amdgcn_readlane((int)v, lane);
}
__device__ __forceinline__ u64 ord_d(double v) {
  const u64 u = (u64)__double_as_longlong(v);
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

// One workgroup a batch entry, one wave a row: the row's sum, then its k best of the chunks' sorted lists (a lane holds
// a list's head): candidates from a bound, ranked all at once; at the end one wave does the same with the rows' lists.
__global__ __launch_bounds__(1024) void beam_pick_kernel(SelArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  u64* sc = reinterpret_cast<u64*>(smem);             // [W][K] ordered bits of the scores, descending
  u64* cand = sc + a.W * a.K + (a.W * a.K + 1) / 2;   // [waves][kSelList]
  int* ti = reinterpret_cast<int*>(sc + a.W * a.K);   // [W][K] tokens; -1 = none
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, nw = blockDim.x >> 6;
  const int b = blockIdx.x, K = a.K;
  const u64 ninf = ord_d(-INFINITY);
  __shared__ unsigned char fin_s[kSelMaxW];
  __shared__ int ci[kSelFew];
  auto put = [&](int w, int i, u64 k, double s, double M, double lt) {  // i-th best of row w
    double v = s + (((double)unord_f((unsigned)(k >> 32)) - M) - lt) + 0.0;
    sc[w * K + i] = ord_d(v);
    ti[w * K + i] = k ? key_idx(k) : -1;
  };
  for (int w = wave; w < a.W; w += nw) {
    const long row = (long)b * a.W + w;
    // everything that the row may need is requested at once; of a row that is out, nothing but the score has been written
    const u64* lp = a.keys + (row * a.C + min(lane, a.C - 1)) * K;
    const unsigned char ended = a.fin ? a.fin[row] : 0;
    const float s = a.score[row];
    const float2 x = a.ml[row * a.C + min(lane, a.C - 1)];
    u64 head = lp[0], nxt[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) nxt[i] = lp[min(i + 1, K - 1)];
    const bool fin = ended != 0;
    if (lane == 0) fin_s[w] = fin;
    double M = 0.0, lt = 0.0;  // the row's maximum, and the log of its sum of e^{x - M}: apart, since M may be huge
    bool live = !fin && fabsf(s) < INFINITY;
    if (live) {
      const float Mf = unord_f(wave_umax(lane < a.C ? ord_f(x.x) : 0u));
      M = (double)Mf;
      // the chunks' weights and their sum in 32 bits, like the terms they sum; its log in 64
      const float t = wave_fsum(lane < a.C && !(x.x == -INFINITY && x.y == 0.f) ? x.y * __expf(x.x - Mf) : 0.f);
      lt = log((double)t);
      live = t > 0.f && lt - lt == 0.0 && M - M == 0.0;  // a row of -inf, or with a NaN or +inf, offers nothing
    }
    if (live) {
      // The row's K best of the chunks' sorted lists, a list a lane. No more than K lists matter, those with the largest
      // heads, and of them the keys from the K-th largest head on; mostly few more than K.
      if (lane >= a.C) head = 0;
#pragma unroll
      for (int i = 0; i < 3; ++i) nxt[i] = lane < a.C && i + 1 < K ? nxt[i] : 0;
      u64* cl = cand + wave * kSelList;
      u64 k[4] = {head, nxt[0], nxt[1], nxt[2]};
      int cnt = 0;
      if (a.C * K <= kSelList) {  // all of them
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          k[i] = lane + 64 * i < a.C * K ? (a.keys + row * a.C * K)[lane + 64 * i] : 0;
          cnt += __popcll(__ballot(k[i] != 0));
        }
      } else {
        const int lists = __popcll(__ballot(head != 0)), q = (K + lists - 1) / lists;
        u64 bar;
        if (q == 1) {
          const unsigned h[1] = {(unsigned)(head >> 32)};
          bar = (u64)kth_below(h, 1, wave_umax(h[0]), K) << 32;
        } else {  // fewer lists than K: the least of their q-th keys has q keys of each list at or above it
          bar = ~wave_kmax(~(lane < a.C && head ? lp[q - 1] : ~0ull));
          if (!bar) bar = 1;
        }
        for (int i = 0; i < K; i += 4) {  // along the lists that reach the bar, four keys at a time
          u64 in = 0;
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            in = __ballot(k[u] >= bar);
            const int at = cnt + __popcll(in & ((1ull << lane) - 1));
            if (k[u] >= bar && at < kSelList) cl[at] = k[u];
            cnt += __popcll(in);
          }
          if (!in) break;
          const bool on = k[3] >= bar;
#pragma unroll
          for (int u = 0; u < 4; ++u) k[u] = on && i + 4 + u < K ? lp[i + 4 + u] : 0;
        }
        wave_fence();
#pragma unroll
        for (int i = 0; i < 4; ++i) k[i] = lane + 64 * i < min(cnt, kSelList) ? cl[lane + 64 * i] : 0;
      }
      if (cnt <= kSelList) {  // closer to K, by the K-th largest value among them; then the rank of each
        unsigned x[4], mx = 0, t = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = (unsigned)(k[i] >> 32);
          mx = max(mx, x[i]);
        }
        if (cnt > 64) t = kth_below(x, 0, wave_umax(mx), K);
        wave_fence();
        cnt = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool in = k[i] && x[i] >= t;
          const u64 m = __ballot(in);
          if (in) cl[cnt + __popcll(m & ((1ull << lane) - 1))] = k[i];
          cnt += __popcll(m);
        }
        wave_fence();
        for (int j = lane; j < cnt; j += 64) {
          const u64 mine = cl[j];
          int r = 0;
#pragma unroll 4
          for (int i = 0; i < cnt; ++i) r += cl[i] > mine;
          if (r < K) put(w, r, mine, (double)s, M, lt);
        }
        if (lane >= cnt && lane < K) put(w, lane, 0, (double)s, M, lt);  // fewer columns than K: the rest stays empty
      } else {  // many equal logits: one by one
        u64 cur = head;
        int at = 1;
        for (int i = 0; i < K; ++i) {
          const u64 best = wave_kmax(cur);
          if (lane == 0) put(w, i, best, (double)s, M, lt);
          if (cur == best && best) { cur = at < K ? lp[at] : 0; ++at; }
        }
      }
    } else {
      // every score is -inf, but the one continuation of a row that has ended: the lowest tokens stand for the rest
      const bool keep = fin && fabsf(s) < INFINITY;
      for (int i = lane; i < K; i += 64) {
        int t = i;
        u64 v = ninf;
        if (keep) {
          if (i == 0) { t = a.pad; v = ord_d((double)s + 0.0); }
          else t = i - 1 < a.pad ? i - 1 : i;
        }
        sc[w * K + i] = v;
        ti[w * K + i] = t < a.V ? t : -1;
      }
    }
  }
  __syncthreads();
  if (wave != 0) return;
  auto write = [&](int r, int i, u64 v) {  // the r-th best: entry i of the rows' lists
    const long o = (long)b * K + r;
    const u64 u = (v >> 63) ? (v & 0x7FFFFFFFFFFFFFFFull) : ~v;
    const int w = i / K, t = ti[i];
    a.score_out[o] = (float)__longlong_as_double((long long)u);
    a.parent[o] = w;
    a.token[o] = t;
    if (a.fin_out) a.fin_out[o] = fin_s[w] || t == a.eos;
  };
  if (a.W * K <= kSelFew) {
    // few entries (8 values a lane, or 2: 0.4 us of 8 rows' 16): those from the K-th largest high word of the scores on, and the rank of each among them; equal scores in
    // the order of the lists, which is that of w * V + t
    auto few = [&](auto nn) {
      constexpr int N = decltype(nn)::value;
      u64 k[N];
      unsigned x[N], mx = 0, t = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int j = lane + 64 * i;
        k[i] = j < a.W * K && ti[j] >= 0 ? sc[j] : 0;  // 0: none (-inf has bits)
        x[i] = (unsigned)(k[i] >> 32);
        mx = max(mx, x[i]);
      }
      if (a.W * K > K + 16) t = kth_below(x, 0, wave_umax(mx), K);
      int cnt = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const bool in = k[i] && x[i] >= t;
        const u64 m = __ballot(in);
        const int to = cnt + __popcll(m & ((1ull << lane) - 1));
        if (in) { cand[to] = k[i]; ci[to] = lane + 64 * i; }
        cnt += __popcll(m);
      }
      wave_fence();
      for (int j = lane; j < cnt; j += 64) {
        const u64 v = cand[j];
        int r = 0;
#pragma unroll 4
        for (int i = 0; i < cnt; ++i) r += cand[i] > v || (cand[i] == v && i < j);
        if (r < K) write(r, ci[j], v);
      }
    };
    if (a.W * K <= 128) few(std::integral_constant<int, 2>());
    else few(std::integral_constant<int, kSelFew / 64>());
    return;
  }
  // The k best of the rows' sorted lists, a list a lane: k rounds of the wave's largest head (its low word among the lanes
  // with the largest high word), ties to the lowest row. A list's next entry is read ahead.
  const int base = min(lane, a.W - 1) * K, end = lane < a.W ? K : 0;
  u64 cur = end && ti[base] >= 0 ? sc[base] : 0;  // 0: none (-inf has bits)
  int at = 0;
  for (int r = 0; r < K; ++r) {
    const int i = base + min(at + 1, K - 1);
    const u64 nxt = at + 1 < end && ti[i] >= 0 ? sc[i] : 0;
    const u64 best = wave_kmax(cur);
    if (!best) break;
    if (lane == (int)__ffsll((long long)__ballot(cur == best)) - 1) {
      write(r, base + at, cur);
      cur = nxt;
      ++at;
    }
  }
}

// ---- slx_beam_reorder: x[o, b, w] = x[o, b, parent[b, w]] -------------------------------------------------------
// A thread takes one column of all `width` rows of a batch entry: every row is loaded before any is stored, so the
// state may be reordered in place, whatever the parents; in place, rows that stay are neither read nor written. Memory bound where
// it is large: 24 x 4 x 8 rows of bf16, the first 16256 of 32768 elements used, in place with half of the rows staying: 6.0 us for 25 MB
// read and written; a table of 8 x 8 rows of 101 numbers 3.6 us, of which a launch takes 2 and the chain parent -> row the rest. Wide
// states pay for a row's parent and address in scalars, which spill from 9 rows on: 2 x 8 / 16 / 32 / 64 rows of 101 numbers
// 2.8 / 4.6 / 9.0 / 17.6 us, 6 x 2 x 8 / 16 / 32 / 64 rows of 32 KB 4.2 / 6.4 / 11.4 / 21.3 (6 .. 50 MB, 4.7 TB/s at the widest).
struct ReorderArgs {
  const char* src; char* dst;
  long s0, s1, sr, d0, d1, dr;  // byte strides: two outer axes and the rows, of source and destination
  int n0, n1, B, W;
  long cols;                    // columns (elements of the access type) of a row
  const int* parent;
  int in_place;
};

template <typename T, int MW>
__global__ __launch_bounds__(256) void beam_reorder_kernel(ReorderArgs a) {
  const long c = (long)blockIdx.x * 256 + threadIdx.x;
  if (c >= a.cols) return;
  const unsigned n = (unsigned)a.n0 * (unsigned)a.n1 * (unsigned)a.B;  // < 2^31
  for (unsigned o = blockIdx.y; o < n; o += gridDim.y) {
    const unsigned q = o / (unsigned)a.B, b = o - q * (unsigned)a.B, i0 = q / (unsigned)a.n1, i1 = q - i0 * (unsigned)a.n1;
    const int* par = a.parent + (long)b * a.W;
    int from[MW];  // all requested before one is looked at
#pragma unroll
    for (int w = 0; w < MW; ++w) from[w] = par[min(w, a.W - 1)];
    const char* sp = a.src + i0 * a.s0 + i1 * a.s1 + (long)b * a.W * a.sr + c * (long)sizeof(T);
    char* dp = a.dst + i0 * a.d0 + i1 * a.d1 + (long)b * a.W * a.dr + c * (long)sizeof(T);
    T v[MW];
    bool mv[MW];
#pragma unroll
    for (int w = 0; w < MW; ++w) {
      mv[w] = w < a.W;
      if (mv[w]) {
        const int p = (unsigned)from[w] < (unsigned)a.W ? from[w] : w;  // no such beam: the row stays
        mv[w] = !(a.in_place && p == w);
        if (mv[w]) v[w] = *reinterpret_cast<const T*>(sp + p * a.sr);
      }
    }
#pragma unroll
    for (int w = 0; w < MW; ++w)
      if (mv[w]) *reinterpret_cast<T*>(dp + w * a.dr) = v[w];
  }
}

template <typename T>
static void reorder_launch(const ReorderArgs& a, hipStream_t st) {
  const long n = (long)a.n0 * a.n1 * a.B;
  const dim3 grid((unsigned)((a.cols + 255) / 256), (unsigned)(n < 65535 ? n : 65535));
  if (a.W <= 4) hipLaunchKernelGGL((beam_reorder_kernel<T, 4>), grid, dim3(256), 0, st, a);
  else if (a.W <= 8) hipLaunchKernelGGL((beam_reorder_kernel<T, 8>), grid, dim3(256), 0, st, a);
  else if (a.W <= 16) hipLaunchKernelGGL((beam_reorder_kernel<T, 16>), grid, dim3(256), 0, st, a);
  else if (a.W <= 32) hipLaunchKernelGGL((beam_reorder_kernel<T, 32>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((beam_reorder_kernel<T, 64>), grid, dim3(256), 0, st, a);
}

static int chunks_of(const slx_beam_select_desc* d) { return (d->vocab + kSelChunk - 1) / kSelChunk; }

static int check_select(const slx_beam_select_desc* d) {
  SLX_CHECK_ARG(d != nullptr, "slx_beam_select: null desc");
  SLX_CHECK_ARG(d->batch >= 0 && d->width > 0 && d->width <= kSelMaxW, "slx_beam_select: 0 <= batch, 0 < width <= %d", kSelMaxW);
  SLX_CHECK_ARG(d->vocab > 0 && d->vocab <= kSelChunk * kSelMaxChunks, "slx_beam_select: 0 < vocab <= %d", kSelChunk * kSelMaxChunks);
  SLX_CHECK_ARG(launch_fits((int64_t)d->batch * d->width * chunks_of(d), 256), "slx_beam_select: batch * width rows of %d chunks of %d must be < 2^24 chunks", chunks_of(d), kSelChunk);
  SLX_CHECK_ARG(d->k > 0 && d->k <= kSelMaxK && d->k <= (int64_t)d->width * d->vocab, "slx_beam_select: 0 < k <= %d and <= width * vocab", kSelMaxK);
  SLX_CHECK_ARG(d->ldx >= d->vocab, "slx_beam_select: ldx >= vocab");
  SLX_CHECK_ARG(!d->finished || (d->pad >= 0 && d->pad < d->vocab), "slx_beam_select: pad outside the vocabulary");
  return 0;
}

}  // namespace slx

using namespace slx;

extern "C" {

int64_t slx_beam_select_ws_bytes(const slx_beam_select_desc* d) {
  if (int rc = check_select(d)) return rc;
  const int64_t C = chunks_of(d);
  return (int64_t)d->batch * d->width * C * (8 + 8 * (int64_t)d->k);
}

int slx_beam_select(const slx_beam_select_desc* d, slx_stream_t s) {
  if (int rc = check_select(d)) return rc;
  if (d->batch == 0) return 0;
  SLX_CHECK_ARG(d->logits && d->score && d->score_out && d->parent && d->token, "slx_beam_select: null argument");
  const int64_t need = slx_beam_select_ws_bytes(d);
  SLX_CHECK_ARG(d->ws && ((uintptr_t)d->ws & 7) == 0 && d->ws_bytes >= need, "slx_beam_select: needs an 8-B aligned workspace of %lld bytes", (long long)need);
  SelArgs a;
  memset(&a, 0, sizeof(a));
  a.x = d->logits; a.ldx = d->ldx; a.score = d->score; a.fin = d->finished;
  a.score_out = d->score_out; a.parent = d->parent; a.token = d->token; a.fin_out = d->finished_out;
  a.B = d->batch; a.W = d->width; a.V = d->vocab; a.K = d->k; a.pad = d->pad; a.eos = d->eos;
  a.C = chunks_of(d);
  a.ml = (float2*)d->ws;
  a.keys = (u64*)((char*)d->ws + (int64_t)a.B * a.W * a.C * 8);
  const dim3 grid((unsigned)((int64_t)a.C * a.B * a.W));
  if (d->logits_bf16) hipLaunchKernelGGL((beam_chunk_kernel<bf16>), grid, dim3(256), 0, (hipStream_t)s, a);
  else hipLaunchKernelGGL((beam_chunk_kernel<float>), grid, dim3(256), 0, (hipStream_t)s, a);
  SLX_LAUNCH_CHECK("slx_beam_select (chunks)");
  const int nw = a.W < 16 ? a.W : 16;
  const int wk = a.W * a.K, lds = 8 * (wk + (wk + 1) / 2) + nw * kSelList * 8;
  if (lds > 60 * 1024) {
    hipError_t e = hipFuncSetAttribute((const void*)beam_pick_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    SLX_CHECK_ARG(e == hipSuccess, "slx_beam_select: %d B of LDS: %s", lds, hipGetErrorString(e));
  }
  hipLaunchKernelGGL(beam_pick_kernel, dim3(a.B), dim3(64 * nw), lds, (hipStream_t)s, a);
  SLX_LAUNCH_CHECK("slx_beam_select");
  return 0;
}

int slx_beam_reorder(const slx_beam_reorder_desc* d, slx_stream_t s) {
  SLX_CHECK_ARG(d != nullptr, "slx_beam_reorder: null desc");
  SLX_CHECK_ARG(d->n0 >= 0 && d->n1 >= 0 && d->batch >= 0 && d->row_bytes >= 0 && d->width > 0 && d->width <= kSelMaxW,
                "slx_beam_reorder: extents >= 0, 0 < width <= %d", kSelMaxW);
  if (d->n0 == 0 || d->n1 == 0 || d->batch == 0 || d->row_bytes == 0) return 0;
  SLX_CHECK_ARG(d->src && d->dst && d->parent, "slx_beam_reorder: null argument");
  ReorderArgs a;
  memset(&a, 0, sizeof(a));
  a.src = (const char*)d->src; a.dst = (char*)d->dst;
  a.s0 = d->s0; a.s1 = d->s1; a.sr = d->src_row; a.d0 = d->d0; a.d1 = d->d1; a.dr = d->dst_row;
  a.n0 = d->n0; a.n1 = d->n1; a.B = d->batch; a.W = d->width; a.parent = d->parent;
  a.in_place = d->src == d->dst;
  SLX_CHECK_ARG(!a.in_place || (a.s0 == a.d0 && a.s1 == a.d1 && a.sr == a.dr), "slx_beam_reorder: in place needs equal strides");
  // the widest access that the row's length and every stride and address allow
  const uint64_t u = (uint64_t)(uintptr_t)d->src | (uint64_t)(uintptr_t)d->dst | (uint64_t)d->s0 | (uint64_t)d->s1 |
                     (uint64_t)d->src_row | (uint64_t)d->d0 | (uint64_t)d->d1 | (uint64_t)d->dst_row | (uint64_t)d->row_bytes;
  const int w = (u & 15) == 0 ? 16 : (u & 3) == 0 ? 4 : (u & 1) == 0 ? 2 : 1;
  a.cols = d->row_bytes / w;
  SLX_CHECK_ARG(launch_fits((a.cols + 255) / 256, 256), "slx_beam_reorder: rows too long");
  SLX_CHECK_ARG((double)d->n0 * d->n1 * d->batch < 2147483648.0, "slx_beam_reorder: n0 * n1 * batch must be < 2^31");
  if (w == 16) reorder_launch<u32x4>(a, (hipStream_t)s);
  else if (w == 4) reorder_launch<unsigned>(a, (hipStream_t)s);
  else if (w == 2) reorder_launch<unsigned short>(a, (hipStream_t)s);
  else reorder_launch<unsigned char>(a, (hipStream_t)s);
  SLX_LAUNCH_CHECK("slx_beam_reorder");
  return 0;
}

}  // extern "C"
