// rope_append.cu — rotation of queries and keys by their positions (lvb_rope) and the append of
// new tokens to the paged KV cache with the rotation on the way (lvb_kv_append).
//
// Both are streams of 16-byte loads and stores with a few operations per element, bound by HBM
// for many tokens and by the latency of one load-store chain for few. A CTA takes a few tokens;
// its threads first work out cos and sin once per (token, pair) into shared memory (the angle
// pos·freq in 64 bits, reduced to a fraction of a turn there: at position 100,000 a 32-bit angle
// has an error of 4e-3 rad), then every thread keeps the cos and sin of its pairs in registers and
// walks over the heads, two 16-byte vectors per head: with halves the two that face each other
// (elements i.. and i+pairs..), with adjacent pairs two neighbouring ones, so either way the
// vectors hold whole pairs and an in-place call is safe.
#include <algorithm>
#include <type_traits>

#include "paged.cuh"

namespace lvb {

namespace {

constexpr int kRotThreads = 256;
constexpr int kRotCtas = 4;           // per SM: 64 registers a thread
constexpr int kRotTokens = 16;        // most tokens per CTA
// Heads that a thread has under way at a time. Two, with four CTAs per SM, against one with five,
// three or four with three: a video clip's gradient 18.3 us against 22.7, 19.8 and 19.9; prompts into
// the cache 14.5 against 15.9, 14.5 and 14.6; 268 MB of Q and K 87.1 against 96.2, 89.0 and 88.9.
constexpr int kRotUnroll = 2;

struct RotArgs {
  int pairs, n_axes, inverse;
  int sec_end[LVB_ROPE_MAX_AXES];     // first pair behind each axis's section
  const double* freqs;
  const int* pos;                     // NULL: the token's place (append)
  long long pos_axis;
};

__device__ __forceinline__ int axis_of(const RotArgs& r, int pair) {
  int a = 0;
#pragma unroll
  for (int i = 0; i < LVB_ROPE_MAX_AXES - 1; ++i) a += (i + 1 < r.n_axes && pair >= r.sec_end[i]);
  return a;
}

// cos and sin of pos·freq: the turn's fraction in 64 bits, then 32-bit functions of half-turns.
__device__ __forceinline__ float2 turn(int pos, double freq, int inverse) {
  const double t = (double)pos * freq * 0.15915494309189533577;   // 1/(2π)
  const float f = (float)(t - rint(t));
  float2 cs;
  sincospif(2.f * f, &cs.y, &cs.x);
  if (inverse) cs.y = -cs.y;
  return cs;
}

template <typename T>
struct Vec {
  static constexpr int N = 16 / (int)sizeof(T);
  __device__ static __forceinline__ void unpack(const uint4& u, float (&f)[N]) {
    if constexpr (std::is_same<T, float>::value) {
      f[0] = __uint_as_float(u.x);
      f[1] = __uint_as_float(u.y);
      f[2] = __uint_as_float(u.z);
      f[3] = __uint_as_float(u.w);
    } else {
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, __half>::value) {
          const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
          f[2 * i] = v.x;
          f[2 * i + 1] = v.y;
        } else {   // a bf16 is the upper half of its fp32
          f[2 * i] = __uint_as_float(w[i] << 16);
          f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
      }
    }
  }
  __device__ static __forceinline__ uint4 pack(const float (&f)[N]) {
    if constexpr (std::is_same<T, float>::value) {
      return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                        __float_as_uint(f[3]));
    } else {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, __half>::value) {
          const __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&v);
        } else {
          const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
      }
      return make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
};

// One thread's N pairs of one head: u and v become the rotated vectors.
template <typename T, bool HALVES>
__device__ __forceinline__ void rotate2(uint4& u, uint4& v, const float (&c)[Vec<T>::N],
                                        const float (&s)[Vec<T>::N]) {
  constexpr int N = Vec<T>::N;
  float a[N], b[N];
  Vec<T>::unpack(u, a);
  Vec<T>::unpack(v, b);
  if constexpr (HALVES) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float x = a[i], y = b[i];
      a[i] = x * c[i] - y * s[i];
      b[i] = y * c[i] + x * s[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float x = a[2 * i], y = a[2 * i + 1], z = b[2 * i], w = b[2 * i + 1];
      a[2 * i] = x * c[i] - y * s[i];
      a[2 * i + 1] = y * c[i] + x * s[i];
      b[2 * i] = z * c[N / 2 + i] - w * s[N / 2 + i];
      b[2 * i + 1] = w * c[N / 2 + i] + z * s[N / 2 + i];
    }
  }
  u = Vec<T>::pack(a);
  v = Vec<T>::pack(b);
}

// A thread's heads h, h + step, ... < h1 of a list of heads (`rows(h)` gives where head h comes from
// and goes to, and whether it turns), two vectors at element offsets o0 and o1 each, kRotUnroll
// heads at a time. The first batch is loaded before the CTA works out its angles and places, so
// that this chain of loads runs beside it.
template <typename T, bool HALVES>
struct HeadWalk {
  uint4 u[kRotUnroll], v[kRotUnroll];
  int h, h1, step, o0, o1;
  template <typename Src>
  __device__ __forceinline__ void load(const Src& src) {
#pragma unroll
    for (int k = 0; k < kRotUnroll; ++k) {
      const int hk = h + k * step;
      if (hk < h1) {
        const T* p = reinterpret_cast<const T*>(src(hk));
        u[k] = *reinterpret_cast<const uint4*>(p + o0);
        v[k] = *reinterpret_cast<const uint4*>(p + o1);
      }
    }
  }
  template <typename Src, typename Dst, typename Turns>
  __device__ __forceinline__ void finish(const Src& src, const Dst& dst, const Turns& turns,
                                         const float (&c)[Vec<T>::N], const float (&s)[Vec<T>::N]) {
    while (true) {
#pragma unroll
      for (int k = 0; k < kRotUnroll; ++k) {
        const int hk = h + k * step;
        if (hk < h1) {
          if (turns(hk)) rotate2<T, HALVES>(u[k], v[k], c, s);
          T* p = reinterpret_cast<T*>(dst(hk));
          *reinterpret_cast<uint4*>(p + o0) = u[k];
          *reinterpret_cast<uint4*>(p + o1) = v[k];
        }
      }
      h += kRotUnroll * step;
      if (h >= h1) break;
      load(src);
    }
  }
};

// A thread's place in its CTA: token i of the CTA's, vector pair j of a head, and the first of
// the heads it walks (step `hpp`).
struct Lane {
  int i, j, hl, hpp;
  bool on;
  __device__ __forceinline__ Lane(int n_tok, int tasks) {
    const int per = n_tok * tasks;
    hpp = kRotThreads / per;
    hl = threadIdx.x / per;
    const int rem = threadIdx.x - hl * per;
    i = rem / tasks;
    j = rem - i * tasks;
    on = hl < hpp;
  }
};

// Element offsets of a thread's two vectors in a head, and whether they turn.
template <typename T, bool HALVES>
__device__ __forceinline__ bool lane_vectors(int j, int pairs, int& o0, int& o1) {
  constexpr int N = Vec<T>::N;
  const bool turns = j * N < pairs;
  if (HALVES && turns) {
    o0 = j * N;
    o1 = pairs + j * N;
  } else {
    o0 = 2 * j * N;     // also the unrotated rest: elements from 2·pairs on, in order
    o1 = o0 + N;
  }
  return turns;
}

template <typename T>
__device__ __forceinline__ void lane_angles(const float2* cs, int i, int j, int pairs, bool turns,
                                            float (&c)[Vec<T>::N], float (&s)[Vec<T>::N]) {
  constexpr int N = Vec<T>::N;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const float2 v = turns ? cs[i * pairs + j * N + k] : make_float2(1.f, 0.f);
    c[k] = v.x;
    s[k] = v.y;
  }
}

// ----------------------------------------------------------------------------------------
// lvb_rope
// ----------------------------------------------------------------------------------------
struct RopeParams {
  RotArgs rot;
  int n_tok, tasks, S, heads_per_cta, Hq, Hkv;
  long long pos_b, pos_s;
  const uint8_t *Q, *K;
  uint8_t *Qo, *Ko;
  long long q[3], k[3], qo[3], ko[3];   // byte strides of batch, head, seq
};

template <typename T, bool HALVES>
__global__ void __launch_bounds__(kRotThreads, kRotCtas) rope_kernel(const RopeParams p) {
  extern __shared__ float2 cs[];      // [n_tok][pairs]
  griddep_wait();
  griddep_launch_dependents();
  const int s0 = blockIdx.x * p.n_tok;
  const int b = blockIdx.z;
  const int pairs = p.rot.pairs;
  const Lane l(p.n_tok, p.tasks);
  const long long s = s0 + l.i;
  const bool on = l.on && s < p.S;
  // The CTA's heads of the list Q heads, K heads.
  const int h0 = blockIdx.y * p.heads_per_cta;
  HeadWalk<T, HALVES> walk;
  const bool turns = lane_vectors<T, HALVES>(l.j, pairs, walk.o0, walk.o1);
  walk.h = h0 + l.hl;
  walk.h1 = on ? min(h0 + p.heads_per_cta, p.Hq + p.Hkv) : 0;
  walk.step = l.hpp;
  const long long qs = b * p.q[0] + s * p.q[2], ks = b * p.k[0] + s * p.k[2];
  const long long qd = b * p.qo[0] + s * p.qo[2], kd = b * p.ko[0] + s * p.ko[2];
  auto src = [&](int h) { return h < p.Hq ? p.Q + qs + h * p.q[1] : p.K + ks + (h - p.Hq) * p.k[1]; };
  auto dst = [&](int h) { return h < p.Hq ? p.Qo + qd + h * p.qo[1] : p.Ko + kd + (h - p.Hq) * p.ko[1]; };
  walk.load(src);
  for (int x = threadIdx.x; x < p.n_tok * pairs; x += kRotThreads) {
    const int i = x / pairs, pr = x - i * pairs;
    if (s0 + i < p.S) {
      const int pos = p.rot.pos[axis_of(p.rot, pr) * p.rot.pos_axis + b * p.pos_b +
                                (s0 + i) * p.pos_s];
      cs[x] = turn(pos, p.rot.freqs[pr], p.rot.inverse);
    }
  }
  __syncthreads();
  if (!on) return;
  float c[Vec<T>::N], sn[Vec<T>::N];
  lane_angles<T>(cs, l.i, l.j, pairs, turns, c, sn);
  walk.finish(src, dst, [&](int) { return turns; }, c, sn);
}

// ----------------------------------------------------------------------------------------
// lvb_kv_append
// ----------------------------------------------------------------------------------------
struct AppendParams {
  RotArgs rot;
  PagedSeqs seqs;
  int n_tok, tasks, T, heads_per_cta, Hq, Hkv;   // Hq 0: no queries
  int check_chunks;                              // of kRotThreads - 32 sequences
  const uint8_t *K, *V, *Q;
  uint8_t *Kc, *Vc, *Qo;
  long long k[2], v[2], q[2], qo[2];             // byte strides of token, head
  long long kc[3], vc[3];                        // of page, slot, head
};

// The sequences of tokens t0 .. t0+n-1 (n <= 32), by one warp: lane i gets token i's and its place in
// the list, -1 for none. The last sequence that starts at or before t0 is found 32 at a time (two
// rounds for 1,024), then 32 sequences from there on are held by the lanes and every token is
// looked up among them: a few dependent loads for all tokens of the CTA (2,000 sequences of one token
// 17.5 us when each token's warp went through the list from its start). Where the offsets are not in
// order a token may be missed; it is never taken for another sequence's.
__device__ __forceinline__ int sequences_of(const PagedSeqs& p, int t0, int n, SeqInfo* s) {
  const int lane = (int)lane_id();
  int b = -1;
  if (!p.cu_q) {
    if (lane < n) {
      b = (t0 + lane) / p.max_q;
      if (b >= p.batch) b = -1;
      else *s = seq_info(p, b);
    }
    return b;
  }
  int lo = 0, left = p.batch;
  while (left > 32) {
    const int step = (left + 31) / 32, k = lo + lane * step;
    const unsigned at = __ballot_sync(0xffffffffu, lane * step < left && p.cu_q[min(k, p.batch)] <= t0);
    const int skip = at ? (31 - __clz(at)) * step : 0;
    lo += skip;
    left = min(step, left - skip);
  }
  int row0 = 0, row1 = 0, len = 0;
  for (; lo < p.batch; lo += 32) {
    const int k = min(lo + lane, p.batch - 1);
    const int w0 = p.cu_q[k], w1 = p.cu_q[k + 1], wl = p.lens[k];
    int src = 0;          // the last of them that starts at or before the lane's token
#pragma unroll
    for (int step = 16; step > 0; step >>= 1) {
      const int start = __shfl_sync(0xffffffffu, w0, src + step);
      if (start <= t0 + lane) src += step;
    }
    const int r0 = __shfl_sync(0xffffffffu, w0, src);
    const int r1 = __shfl_sync(0xffffffffu, w1, src);
    const int l = __shfl_sync(0xffffffffu, wl, src);
    if (lane < n && b < 0 && r0 <= t0 + lane && t0 + lane < r1) {
      b = min(lo + src, p.batch - 1);
      row0 = r0;
      row1 = r1;
      len = l;
    }
    if (!__any_sync(0xffffffffu, lane < n && b < 0)) break;
  }
  if (b >= 0) *s = seq_checked(p, b, len, row0, row1);
  return b;
}

template <typename T, bool HALVES>
__global__ void __launch_bounds__(kRotThreads, kRotCtas) append_kernel(const AppendParams p) {
  extern __shared__ float2 cs[];      // [n_tok][pairs]
  __shared__ long long sh_k[kRotTokens], sh_v[kRotTokens];   // cache rows, bytes; -1: left out
  __shared__ int sh_place[kRotTokens];
  griddep_wait();
  griddep_launch_dependents();
  const int t0 = blockIdx.x * p.n_tok;
  const int pairs = p.rot.pairs;
  const Lane l(p.n_tok, p.tasks);
  const long long t = t0 + l.i;
  // The CTA's heads of the list Q heads, K heads, V heads.
  const int h0 = blockIdx.y * p.heads_per_cta;
  HeadWalk<T, HALVES> walk;
  const bool turns = lane_vectors<T, HALVES>(l.j, pairs, walk.o0, walk.o1);
  walk.h = h0 + l.hl;
  walk.h1 = l.on && t < p.T ? min(h0 + p.heads_per_cta, p.Hq + 2 * p.Hkv) : 0;
  walk.step = l.hpp;
  const int hk0 = p.Hq, hv0 = p.Hq + p.Hkv;     // the first K and V heads of the list
  auto src = [&](int h) {
    return h < hk0 ? p.Q + t * p.q[0] + h * p.q[1]
                   : h < hv0 ? p.K + t * p.k[0] + (h - hk0) * p.k[1]
                             : p.V + t * p.v[0] + (h - hv0) * p.v[1];
  };
  walk.load(src);
  // One warp looks up the tokens' places; the others, when the positions are given, work out the
  // angles meanwhile. Positions that count the places have to wait for them.
  auto angles = [&](int first, int step) {
    for (int x = first; x < p.n_tok * pairs; x += step) {
      const int i = x / pairs, pr = x - i * pairs;
      if (t0 + i < p.T) {
        const int pos = p.rot.pos ? p.rot.pos[axis_of(p.rot, pr) * p.rot.pos_axis + t0 + i]
                                  : p.seqs.prefix_len + max(sh_place[i], 0);
        cs[x] = turn(pos, p.rot.freqs[pr], p.rot.inverse);
      }
    }
  };
  if (threadIdx.x >= 32) {
    if (p.rot.pos) angles(threadIdx.x - 32, kRotThreads - 32);
    // Every sequence's entries are checked by some thread, so that wrong ones are reported for a
    // sequence without new rows too, and where the search for a token's sequence is led astray.
    if (blockIdx.y == 0)
      for (int c = blockIdx.x; c < p.check_chunks; c += gridDim.x) {
        const unsigned b = (unsigned)c * (kRotThreads - 32) + threadIdx.x - 32;
        if (b < (unsigned)p.seqs.batch) seq_info(p.seqs, (int)b);
      }
  } else {
    const int i = threadIdx.x, n = min(p.n_tok, p.T - t0);
    SeqInfo s{0, 0, 0};
    const int b = sequences_of(p.seqs, t0, n, &s);
    if (i < n) {
      // (a sequence whose rows do not fit has none)
      int place = b >= 0 && t0 + i - s.tok0 < s.qlen ? s.len - s.qlen + (t0 + i - s.tok0) : -1;
      if (place >= 0) {
        const int pi = place / p.seqs.page_size;
        const int page = p.seqs.table[b * p.seqs.table_stride + pi];
        if (page < 0 || page >= p.seqs.num_pages) {
          report_bad(p.seqs.status, kBadPage, b);
          place = -1;
        } else {
          const int slot = place - pi * p.seqs.page_size;
          sh_k[i] = page * p.kc[0] + slot * p.kc[1];
          sh_v[i] = page * p.vc[0] + slot * p.vc[1];
        }
      }
      sh_place[i] = place;
    }
  }
  __syncthreads();
  if (!p.rot.pos && pairs) {
    angles(threadIdx.x, kRotThreads);
    __syncthreads();
  }
  if (!l.on || t >= p.T || sh_place[l.i] < 0) return;
  float c[Vec<T>::N], sn[Vec<T>::N];
  lane_angles<T>(cs, l.i, l.j, pairs, turns, c, sn);
  uint8_t* kc = p.Kc + sh_k[l.i];
  uint8_t* vc = p.Vc + sh_v[l.i];
  auto dst = [&](int h) {
    return h < hk0 ? p.Qo + t * p.qo[0] + h * p.qo[1]
                   : h < hv0 ? kc + (h - hk0) * p.kc[2] : vc + (h - hv0) * p.vc[2];
  };
  walk.finish(src, dst, [&](int h) { return turns && h < hv0; }, c, sn);
}

// Tokens per CTA and heads per CTA. As many tokens as leave about three CTAs per SM (the angles of a
// token are worked out once for all its heads, 768 per CTA; the video clip's gradient 18.6 us with
// 16 tokens, 20.0 with 8, 22.1 with 4). Up to half more CTAs than run at once would wait for a second
// round of few: then as many tokens as make one full round (4,900 tokens of 48 128-wide heads in 545 CTAs of
// 9 tokens 24.8 us, in 613 of 8 29.8), or, at the most tokens and when a CTA's bytes take longer than its
// chain of loads (3 us to the first, 1 us per kRotUnroll heads), two full rounds (10,000 such tokens in
// 1,112 CTAs of 9 46.7, in 625 of 16 55.7; but two times 5,000 positions of eight 64-wide heads, whose
// chain is longer, 9.1 and 7.3). When one token per CTA is too few, its heads are split too, never
// below one pass of the CTA's threads.
void rot_grid(long long tokens_per_row, long long rows, int heads, int tasks, int sms, int* n_tok,
              int* heads_per_cta) {
  const long long slots = (long long)kRotCtas * sms;
  auto ctas = [&](int n) { return rows * ((tokens_per_row + n - 1) / n); };
  int n = 1;
  while (2 * n <= kRotTokens && 2 * n * tasks <= kRotThreads && ctas(2 * n) >= 3LL * sms) n *= 2;
  if (ctas(n) > slots && 2 * ctas(n) < 3 * slots) {
    while (ctas(n) > slots && n < kRotTokens && (n + 1) * tasks <= kRotThreads) ++n;
    const int steps = heads * n * tasks / (kRotThreads * kRotUnroll);
    const double bytes_us = n * heads * tasks * 64.0 * (double)slots / 6.5e6;
    if (ctas(n) > slots && bytes_us > 3.0 + steps) {
      while (n > 1 && ctas(n - 1) <= 2 * slots) --n;
    }
  }
  const int hpp = std::max(1, kRotThreads / (n * tasks));
  const long long split = std::max<long long>(1, slots / ctas(n));
  int per = (int)((heads + split - 1) / split);
  per = std::min(heads, (per + hpp - 1) / hpp * hpp);
  *n_tok = n;
  *heads_per_cta = std::max(1, per);
}

void fill_rot(RotArgs* r, const lvb_rotation& rot, const int32_t* pos, const double* freqs,
              long long pos_axis) {
  r->pairs = rot.pairs;
  r->n_axes = rot.n_axes;
  r->inverse = rot.inverse ? 1 : 0;
  int end = 0;
  for (int a = 0; a < LVB_ROPE_MAX_AXES; ++a) {
    end += a < rot.n_axes ? rot.sections[a] : 0;
    r->sec_end[a] = end;
  }
  r->freqs = freqs;
  r->pos = pos;
  r->pos_axis = pos_axis;
}

}  // namespace

int rope_launch(const lvb_rope_desc* d, const long long qs[3], const long long ks[3],
                const long long qos[3], const long long kos[3], const void* Q, const void* K,
                void* Qo, void* Ko, const int32_t* pos, const double* freqs, cudaStream_t stream,
                DeviceState* dev) {
  const char* op = "lvb_rope";
  const int es = dtype_size(d->dtype);
  RopeParams p = {};
  fill_rot(&p.rot, d->rot, pos, freqs, d->pos_stride[0]);
  p.pos_b = d->pos_stride[1];
  p.pos_s = d->pos_stride[2];
  p.S = (int)d->seq;
  p.Hq = (int)d->heads_q;
  p.Hkv = (int)d->heads_kv;
  p.tasks = (int)d->head_dim * es / 32;
  p.Q = (const uint8_t*)Q;
  p.K = (const uint8_t*)K;
  p.Qo = (uint8_t*)Qo;
  p.Ko = (uint8_t*)Ko;
  for (int i = 0; i < 3; ++i) {
    p.q[i] = qs[i] * es;
    p.k[i] = ks[i] * es;
    p.qo[i] = qos[i] * es;
    p.ko[i] = kos[i] * es;
  }
  const int heads = p.Hq + p.Hkv;
  rot_grid(d->seq, d->batch, heads, p.tasks, dev->sm_count, &p.n_tok, &p.heads_per_cta);
  const dim3 grid((unsigned)((d->seq + p.n_tok - 1) / p.n_tok),
                  (unsigned)((heads + p.heads_per_cta - 1) / p.heads_per_cta), (unsigned)d->batch);
  const size_t smem = (size_t)p.n_tok * p.rot.pairs * sizeof(float2);
  const bool halves = d->rot.layout == LVB_ROPE_HALVES;
  SmemAttr none;
  auto go = [&](auto kern) {
    return launch_serial(op, kern, none, dev, grid, kRotThreads, smem, stream, p);
  };
  if (d->dtype == LVB_F32) return go(halves ? rope_kernel<float, true> : rope_kernel<float, false>);
  if (d->dtype == LVB_F16) return go(halves ? rope_kernel<__half, true> : rope_kernel<__half, false>);
  return go(halves ? rope_kernel<__nv_bfloat16, true> : rope_kernel<__nv_bfloat16, false>);
}

int append_launch(const lvb_append_desc* d, const PagedLayout& lay, const long long ks[2],
                  const long long vs[2], void* Kc, void* Vc, const void* K, const void* V,
                  const void* Q, void* Qo, const int32_t* table, const int32_t* seq_lens,
                  const int32_t* cu_q, const int32_t* pos, const double* freqs, cudaStream_t stream,
                  DeviceState* dev) {
  const char* op = "lvb_kv_append";
  const lvb_paged_desc& g = d->paged;
  AppendParams p = {};
  fill_rot(&p.rot, d->rot, pos, freqs, d->pos_stride);
  paged_seqs(&p.seqs, g, table, seq_lens, cu_q, nullptr, dev);
  p.T = (int)g.tokens;
  p.check_chunks = (int)((g.batch + kRotThreads - 33) / (kRotThreads - 32));
  p.Hq = Q ? (int)g.heads_q : 0;
  p.Hkv = (int)g.heads_kv;
  p.tasks = (int)g.head_dim * 2 / 32;
  p.K = (const uint8_t*)K;
  p.V = (const uint8_t*)V;
  p.Q = (const uint8_t*)Q;
  p.Kc = (uint8_t*)Kc;
  p.Vc = (uint8_t*)Vc;
  p.Qo = (uint8_t*)Qo;
  for (int i = 0; i < 2; ++i) {
    p.k[i] = ks[i] * 2;
    p.v[i] = vs[i] * 2;
    p.q[i] = lay.q[i] * 2;
    p.qo[i] = lay.o[i] * 2;
  }
  for (int i = 0; i < 3; ++i) {
    p.kc[i] = lay.kc[i] * 2;
    p.vc[i] = lay.vc[i] * 2;
  }
  const int heads = p.Hq + 2 * p.Hkv;
  rot_grid(g.tokens, 1, heads, p.tasks, dev->sm_count, &p.n_tok, &p.heads_per_cta);
  const dim3 grid((unsigned)((g.tokens + p.n_tok - 1) / p.n_tok),
                  (unsigned)((heads + p.heads_per_cta - 1) / p.heads_per_cta));
  const size_t smem = (size_t)p.n_tok * p.rot.pairs * sizeof(float2);
  const bool halves = d->rot.layout == LVB_ROPE_HALVES;
  SmemAttr none;
  auto go = [&](auto kern) {
    return launch_serial(op, kern, none, dev, grid, kRotThreads, smem, stream, p);
  };
  if (g.dtype == LVB_F16) return go(halves ? append_kernel<__half, true> : append_kernel<__half, false>);
  return go(halves ? append_kernel<__nv_bfloat16, true> : append_kernel<__nv_bfloat16, false>);
}

}  // namespace lvb
