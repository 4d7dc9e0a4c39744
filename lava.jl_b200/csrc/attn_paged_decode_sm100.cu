// attn_paged_decode_sm100.cu — attention of few query rows per KV head (group·max_q <= 32) over
// the paged KV cache, B200 (sm_100a).
//
// O = softmax(scale·Q·Kᵀ + mask)·V with one pass over the keys: S of a 128-key block, a running
// reference maximum m per row, p = 2^(s·log2e - m), O += P·V, l += Σp. The cache is read once at
// HBM speed, and the products are turned so that the keys fill the tensor core's 128 rows:
//   Sᵀ (128 keys × NR rows) = K_j·Qᵀ,   Oᵀ (D × NR) += V_jᵀ·P_jᵀ,   NR = 16 or 32 rows
// (rows = position·group + head of the group). P is rounded to the cache's type for the second
// product (the tensor core takes both operands in one 16-bit type); l sums the unrounded p.
//
//   * the 128-key blocks of all (sequence, KV head) items, one after the other, are dealt to the
//     CTAs in equal contiguous runs, so lengths from one key to the whole cache load the SMs
//     evenly. The lengths are on the device: every CTA sums the block counts itself. An item that
//     a run boundary cuts leaves pieces (O, m, l in 32 bits) in the workspace, at most two per
//     CTA, and the join kernel adds them in a fixed order; an item inside a run stores its result;
//   * 192 threads: warp 4 brings Q and the K and V blocks (a box of slots per page and lane)
//     through a ring that runs ahead across items and publishes the items; warp 5 issues the
//     products (QK_j, then PV_{j-1}); warps 0-3 do the softmax (thread = key) and the epilogue
//     (thread = head-dim element);
//   * m of a row moves only when a score exceeds it by 2^8 (p stays <= 256): a block whose scores
//     all stay below needs no row maximum, only one vote over the 128 threads. In fp16 the
//     exponent is shifted by 2^6, away from the subnormals (p <= 2^14).
#include <algorithm>
#include <cmath>

#include "paged.cuh"

namespace lvb {

namespace {

constexpr int kThreads = 192;
constexpr int kTmaWarp = 4;
constexpr int kMmaWarp = 5;
constexpr int kQueue = 4;                  // items published ahead
constexpr int kChunk = 128 * 128;          // one 64-element chunk of a 128-key block
constexpr float kLazy = 8.f;               // log2 units a score may exceed the reference maximum

struct DecParams {
  PagedSeqs seqs;
  int Hq, Hkv, group, nrows, causal, box, keep_parts;
  float scale_log2;
  void* O;
  long long o_st, o_sh;
  float* lse;
  float* part_o;            // [slot][NR][D]
  float* part_ml;           // [slot][NR][2]
  int4* tab;                // [batch·Hkv]
  unsigned long long timeout_ns;
};

template <int D, int NR>
struct Cfg {
  static constexpr int kCh = D / 64;
  static constexpr int kBlock = kCh * kChunk;
  static constexpr int kRing = D == 128 ? 6 : 12;
  static constexpr int kQ = kCh * NR * 128;            // Q of an item
  static constexpr int kP = 2 * NR * 128;              // P of a block: two 64-key chunks
  static constexpr int kTmemCols = NR == 16 ? 64 : 128;
  static constexpr int kSmem = kRing * kBlock + 2 * kQ + 2 * kP + 4 * NR * 4 + 1024 + 1024;
};

// What the roles need of an item (a run of key blocks of one sequence and KV head).
struct Item {
  int hk, kb0, nblk;        // KV head, first block, blocks
  int len, qlen, tok0;
  int slot;                 // where its piece goes; -1: the whole item, O is stored
  int last;                 // 1: no item, the CTA is done
};

template <bool BF16>
__device__ __forceinline__ uint16_t bits16(float v) {
  if constexpr (BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(v));
  else return __half_as_ushort(__float2half_rn(v));
}

template <int N>
__device__ __forceinline__ void ld_cols(uint32_t taddr, uint32_t (&r)[N]) {
  if constexpr (N == 1) tmem_ld1(taddr, r);
  else if constexpr (N == 4) tmem_ld4(taddr, r);
  else if constexpr (N == 8) tmem_ld8(taddr, r);
  else if constexpr (N == 16) tmem_ld16(taddr, r);
  else tmem_ld32(taddr, r);
}
template <int N>
__device__ __forceinline__ void st_cols(uint32_t taddr, uint32_t (&r)[N]) {
  if constexpr (N == 1) tmem_st1(taddr, r);
  else if constexpr (N == 4) tmem_st4(taddr, r);
  else if constexpr (N == 8) tmem_st8(taddr, r);
  else if constexpr (N == 16) tmem_st16(taddr, r);
  else tmem_st32(taddr, r);
}

__device__ __forceinline__ void drain_wait(uint64_t* bar, uint32_t parity, uint64_t timeout_ns) {
  const uint32_t a = smem_u32(bar);
  const uint64_t t0 = global_ns();
  while (!bar_try_wait(a, parity)) {
    if (global_ns() - t0 > timeout_ns) return;
  }
}

// Whether `pred` holds for any of the 128 softmax threads (barrier 1).
__device__ __forceinline__ bool vote_any(bool pred) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"((uint32_t)pred)
      : "memory");
  return any != 0;
}

// Key blocks of a sequence (0 when it has no query rows).
__device__ __forceinline__ int blocks_of(const SeqInfo& s) {
  return s.qlen > 0 ? (s.len + 127) >> 7 : 0;
}

// RR <= NR: the rows that the softmax works on (the smallest of 1, 4, 8, 16, 32 that holds the
// query rows); the products' other columns are computed and never read.
template <int D, int NR, int RR, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
    paged_decode_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                        const __grid_constant__ CUtensorMap tmV, const DecParams p) {
  using C = Cfg<D, NR>;
  constexpr int R = C::kRing;
  constexpr uint32_t kFmt = BF16 ? 1 : 0;
  constexpr uint32_t kIdescQK = make_idesc(1, kFmt, kFmt, 0, 0, 128, NR);
  constexpr uint32_t kIdescPV = make_idesc(1, kFmt, kFmt, 1, 0, 128, NR);
  constexpr float kShift = BF16 ? 0.f : 6.f;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_1024(smem_raw);
  uint8_t* sRing = smem;                                  // [R][D/64 chunks][128 keys][128 B]
  uint8_t* sQ = sRing + R * C::kBlock;                    // [2][D/64 chunks][NR rows][128 B]
  uint8_t* sP = sQ + 2 * C::kQ;                           // [2][2 chunks][NR rows][128 B]
  float* sRed = reinterpret_cast<float*>(sP + 2 * C::kP); // [4 warps][NR]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sRed + 4 * NR);
  uint64_t* kv_full = bars;              // [R]
  uint64_t* kv_empty = kv_full + R;      // [R]
  uint64_t* q_full = kv_empty + R;       // [2]
  uint64_t* q_empty = q_full + 2;        // [2]
  uint64_t* s_full = q_empty + 2;        // [2]
  uint64_t* s_empty = s_full + 2;        // [2] (128 arrivals)
  uint64_t* p_full = s_empty + 2;        // [2] (128 arrivals)
  uint64_t* p_empty = p_full + 2;        // [2]
  uint64_t* o_full = p_empty + 2;        // an item's last PV done
  uint64_t* o_empty = o_full + 1;        // its epilogue has read Oᵀ (128 arrivals)
  uint64_t* i_full = o_empty + 1;        // [kQueue] item published
  uint64_t* i_empty = i_full + kQueue;   // [kQueue] read by the MMA warp and four softmax warps
  uint64_t* drain = i_empty + kQueue;
  Item* items = reinterpret_cast<Item*>(drain + 1);       // [kQueue]
  long long* sScan = reinterpret_cast<long long*>(items + kQueue);   // [8]: warp sums, then
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sScan + 8);      // the start's offset and b
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const uint32_t warp = warp_id();
  const uint32_t lane = lane_id();
  const int G = gridDim.x;

  if (threadIdx.x == 0) {
    for (int s = 0; s < R; ++s) {
      bar_init(&kv_full[s], 1);
      bar_init(&kv_empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      bar_init(&q_full[i], 1);
      bar_init(&q_empty[i], 1);
      bar_init(&s_full[i], 1);
      bar_init(&s_empty[i], 128);
      bar_init(&p_full[i], 128);
      bar_init(&p_empty[i], 1);
    }
    bar_init(o_full, 1);
    bar_init(o_empty, 128);
    for (int i = 0; i < kQueue; ++i) {
      bar_init(&i_full[i], 1);
      bar_init(&i_empty[i], 5);
    }
    bar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }

  // ---------------- this CTA's run of blocks ----------------
  // Thread i sums the blocks of sequences [i·per, (i+1)·per); a scan over the threads gives the
  // total and the thread whose sequences hold the run's first block.
  const int batch = p.seqs.batch;
  const int per = (batch + kThreads - 1) / kThreads;
  const int sb0 = min((int)threadIdx.x * per, batch), sb1 = min(sb0 + per, batch);
  long long mine = 0;
  for (int b = sb0; b < sb1; ++b) mine += blocks_of(seq_info(p.seqs, b));
  mine *= p.Hkv;
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, incl, o);
    if ((int)lane >= o) incl += v;
  }
  if (lane == 31) sScan[warp] = incl;
  __syncthreads();
  long long before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < (int)warp) before += sScan[w];
    total += sScan[w];
  }
  const long long share = max(1LL, (total + G - 1) / G);
  const long long u0 = blockIdx.x * share;
  const long long u1 = min(u0 + share, total);
  const long long first = before + incl - mine;
  __syncthreads();
  if (u0 < total && u0 >= first && u0 < first + mine) {
    long long off = first;
    for (int b = sb0; b < sb1; ++b) {
      const long long n = (long long)blocks_of(seq_info(p.seqs, b)) * p.Hkv;
      if (u0 < off + n) {
        sScan[0] = off;
        sScan[1] = b;
        break;
      }
      off += n;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tS = tmem;                 // Sᵀ buffers: columns [0, NR) and [NR, 2NR)
  const uint32_t tO = tmem + 2 * NR;        // Oᵀ: columns [2NR, 3NR)
  const WaitGuard g{p.seqs.status, abort_flag, p.timeout_ns};

  if (warp == kTmaWarp) {
    // ---------------- producer: items, Q, K and V blocks ----------------
    if (lane == 0) {
      tma_prefetch_desc(&tmQ);
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
    }
    const BlockLane<D> bl((int)lane, p.box);
    int n = 0;        // ring slots filled
    int it = 0;       // items published
    bool ok = true;
    long long u = u0;
    int base = 0;     // the lanes hold sequences base .. base+31
    SeqInfo sq{0, 0, 0};
    int nb_lane = 0;
    long long off = 0;
    int b = 0;
    if (u < u1) {
      off = sScan[0];
      b = (int)sScan[1];
      base = b & ~31;
      if (base + (int)lane < batch) sq = seq_info(p.seqs, base + lane);
      nb_lane = blocks_of(sq);
    }
    while (u < u1 && ok) {
      // the sequence of block u: the next one with blocks once the current one is passed
      int nb = __shfl_sync(0xffffffffu, nb_lane, b - base);
      if (u >= off + (long long)nb * p.Hkv) {
        off += (long long)nb * p.Hkv;
        int from = b + 1 - base;
        while (true) {
          const unsigned some = from < 32 ? __ballot_sync(0xffffffffu, nb_lane > 0) >> from : 0u;
          if (some) {
            b = base + from + __ffs(some) - 1;
            break;
          }
          base += 32;      // u < total: a later sequence has blocks
          from = 0;
          sq = SeqInfo{0, 0, 0};
          if (base + (int)lane < batch) sq = seq_info(p.seqs, base + lane);
          nb_lane = blocks_of(sq);
        }
        nb = __shfl_sync(0xffffffffu, nb_lane, b - base);
      }
      const int len = __shfl_sync(0xffffffffu, sq.len, b - base);
      const int qlen = __shfl_sync(0xffffffffu, sq.qlen, b - base);
      const int tok0 = __shfl_sync(0xffffffffu, sq.tok0, b - base);
      const int hk = (int)((u - off) / nb);
      const long long o_item = off + (long long)hk * nb;   // the item's first block
      const int kb0 = (int)(u - o_item);
      const int nblk = (int)min((long long)(nb - kb0), u1 - u);
      const bool whole = nblk == nb;
      const int id = b * p.Hkv + hk;
      int slot = -1;
      if (!whole) slot = 2 * blockIdx.x + (u == u0 ? 0 : 1);
      else if (p.keep_parts) slot = 2 * G + id;
      if (kb0 == 0 && lane == 0) {
        const int c1 = (int)((o_item + nb - 1) / share);
        p.tab[id] = make_int4(slot, blockIdx.x + 1, c1,
                              whole && !p.keep_parts ? kItemDone : kItemPieces);
      }
      const int qi = it % kQueue;
      if (!wait_bar_warp(&i_empty[qi], (uint32_t)((it / kQueue) & 1) ^ 1, g, 70, it)) { ok = false; break; }
      if (lane == 0) {
        items[qi] = Item{hk, kb0, nblk, len, qlen, tok0, slot, 0};
        bar_arrive(&i_full[qi]);
      }
      const int qb = it & 1;
      if (!wait_bar_warp(&q_empty[qb], (uint32_t)((it >> 1) & 1) ^ 1, g, 51, it)) { ok = false; break; }
      if (lane == 0) {
        bar_arrive_expect_tx(&q_full[qb], C::kCh * p.nrows * 128);
        for (int c = 0; c < C::kCh; ++c)
          tma_load_3d(sQ + qb * C::kQ + c * NR * 128, &tmQ, c * 64, hk * p.group, tok0, &q_full[qb]);
      }
      ++it;
      const int* row = p.seqs.table + b * p.seqs.table_stride;
      BoxAt at = box_at(bl, row, kb0, len, p.box, p.seqs);
      for (int kb = kb0; kb < kb0 + nblk && ok; ++kb) {
        // the next block's page numbers are on their way while this one's slots are waited for
        BoxAt next{-1, 0};
        if (kb + 1 < kb0 + nblk) next = box_at(bl, row, kb + 1, len, p.box, p.seqs);
        for (int v = 0; v < 2; ++v, ++n) {
          const int s = n % R;
          if (!wait_bar_warp(&kv_empty[s], (uint32_t)((n / R) & 1) ^ 1, g, 52, n)) { ok = false; break; }
          load_block<D>(sRing + s * C::kBlock, v ? &tmV : &tmK, bl, at, p.box, hk, &kv_full[s]);
        }
        at = next;
      }
      u += nblk;
    }
    if (ok) {
      const int qi = it % kQueue;
      if (wait_bar_warp(&i_empty[qi], (uint32_t)((it / kQueue) & 1) ^ 1, g, 70, it) && lane == 0) {
        items[qi].last = 1;
        bar_arrive(&i_full[qi]);
      }
    } else if (lane == 0) {
      // Let the copies in flight land before the CTA's shared memory goes away.
      for (int i = max(0, n - R); i < n; ++i)
        drain_wait(&kv_full[i % R], (uint32_t)((i / R) & 1), p.timeout_ns);
      for (int i = max(0, it - 2); i < it; ++i)
        drain_wait(&q_full[i & 1], (uint32_t)((i >> 1) & 1), p.timeout_ns);
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    // ---------------- MMA issuer: the warp waits, one elected lane issues ----------------
    const uint32_t r_base = smem_u32(sRing);
    const uint32_t q_base = smem_u32(sQ);
    const uint32_t p_base = smem_u32(sP);
    int n_ring = 0;   // ring slots before this item
    int gb = 0;       // blocks before this item
    bool ok = true;
    for (int it = 0; ok; ++it) {
      const int qi = it % kQueue;
      if (!wait_bar_warp(&i_full[qi], (uint32_t)((it / kQueue) & 1), g, 71, it)) break;
      const Item im = items[qi];
      __syncwarp();
      if (lane == 0) bar_arrive(&i_empty[qi]);
      if (im.last) break;
      const int nb = im.nblk;
      const int qb = it & 1;
      if (!wait_bar_warp(&q_full[qb], (uint32_t)((it >> 1) & 1), g, 53, it)) break;
      for (int j = 0; j <= nb && ok; ++j) {
        if (j < nb) {
          const int gj = gb + j;
          const int nk = n_ring + 2 * j;
          const int sk = nk % R;
          if (!wait_bar_warp(&kv_full[sk], (uint32_t)((nk / R) & 1), g, 54, nk)) { ok = false; break; }
          if (!wait_bar_warp(&s_empty[gj & 1], (uint32_t)((gj >> 1) & 1) ^ 1, g, 55, gj)) { ok = false; break; }
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t o = (kk >> 2) * kChunk + (kk & 3) * 32;
            const uint64_t ad = sdesc_sw128(r_base + sk * C::kBlock + o, 16, 1024);
            const uint64_t bd = sdesc_sw128(q_base + qb * C::kQ + (kk >> 2) * NR * 128 +
                                                (kk & 3) * 32, 16, 1024);
            if (elect_one()) mma_f16_ss(tS + NR * (gj & 1), ad, bd, kIdescQK, kk > 0 ? 1u : 0u);
          }
          if (elect_one()) {
            mma_commit(&s_full[gj & 1]);
            mma_commit(&kv_empty[sk]);                   // K_j read
            if (j == nb - 1) mma_commit(&q_empty[qb]);   // the item's Q read for the last time
          }
          __syncwarp();
        }
        if (j > 0) {
          const int gp = gb + j - 1;
          const int nv = n_ring + 2 * (j - 1) + 1;
          const int sv = nv % R;
          const int pb = gp & 1;
          if (!wait_bar_warp(&kv_full[sv], (uint32_t)((nv / R) & 1), g, 56, nv)) { ok = false; break; }
          const int valid = im.len - (im.kb0 + j - 1) * 128;
          if (valid < 128) zero_tail<D>(r_base + sv * C::kBlock, valid);
          if (!wait_bar_warp(&p_full[pb], (uint32_t)((gp >> 1) & 1), g, 57, gp)) { ok = false; break; }
          if (j == 1 && it > 0) {
            // Oᵀ of the previous item read by its epilogue before the first PV overwrites it.
            if (!wait_bar_warp(o_empty, (uint32_t)((it - 1) & 1), g, 58, it)) { ok = false; break; }
          }
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {   // 16 keys per MMA
            // 64-wide heads: the second 64 of the 128 rows read the same chunk again (leading
            // offset 0) and are never looked at.
            const uint64_t ad = sdesc_sw128(r_base + sv * C::kBlock + kk * 16 * 128,
                                            D == 128 ? kChunk : 0, 1024);
            const uint64_t bd = sdesc_sw128(p_base + pb * C::kP + (kk >> 2) * NR * 128 + (kk & 3) * 32, 16, 1024);
            if (elect_one()) mma_f16_ss(tO, ad, bd, kIdescPV, (j == 1 && kk == 0) ? 0u : 1u);
          }
          if (elect_one()) {
            mma_commit(&p_empty[pb]);
            mma_commit(&kv_empty[sv]);                   // V_{j-1} read
            if (j == nb) mma_commit(o_full);
          }
          __syncwarp();
        }
      }
      n_ring += 2 * nb;
      gb += nb;
    }
    if (elect_one()) mma_commit(drain);
    __syncwarp();
    drain_wait(drain, 0, p.timeout_ns);
  } else {
    // ---------------- softmax and epilogue: warps 0-3 ----------------
    const int t = (int)(warp * 32 + lane);              // key within the block / Oᵀ lane (d)
    const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
    const float NEG_INF = -INFINITY;
    const float sl = p.scale_log2;

    // Sequences without a key: zero rows (or no part for the join).
    for (int b = blockIdx.x; b < batch; b += G) {
      const SeqInfo s = seq_info(p.seqs, b);
      if (blocks_of(s) > 0) continue;
      const bool rows = s.qlen > 0;
      for (int hk = t; hk < p.Hkv; hk += 128)
        p.tab[b * p.Hkv + hk] = make_int4(0, 0, -1, rows && p.keep_parts ? kItemNoKeys : kItemDone);
      if (rows && !p.keep_parts) {
        for (int i = 0; i < s.qlen; ++i)
          for (int h = 0; h < p.Hq; ++h) {
            uint16_t* o = reinterpret_cast<uint16_t*>(p.O) + (long long)(s.tok0 + i) * p.o_st + h * p.o_sh;
            if (t < D) o[t] = 0;
            if (p.lse && t == 0) p.lse[(long long)(s.tok0 + i) * p.Hq + h] = NEG_INF;
          }
      }
    }

    int gb = 0;
    for (int it = 0;; ++it) {
      const int qi = it % kQueue;
      // A wait that gave up leaves the CTA's abort flag up; every thread sees it at its next
      // wait, and all 128 leave together after a vote.
      bool ok = wait_bar(&i_full[qi], (uint32_t)((it / kQueue) & 1), g, 72, it);
      if (vote_any(!ok)) break;
      const Item im = items[qi];
      __syncwarp();
      if (lane == 0) bar_arrive(&i_empty[qi]);
      if (im.last) break;
      // Row r = position·group + head of the group; its last visible key.
      int last_key[RR];
#pragma unroll
      for (int r = 0; r < RR; ++r) {
        const int pos = r / p.group;
        last_key[r] = r < p.nrows && pos < im.qlen ? (p.causal ? im.len - im.qlen + pos : im.len - 1) : -1;
      }
      float m_ref[RR], l_part[RR];
#pragma unroll
      for (int r = 0; r < RR; ++r) {
        m_ref[r] = NEG_INF;
        l_part[r] = 0.f;
      }
      for (int j = 0; j < im.nblk; ++j, ++gb) {
        const int key = (im.kb0 + j) * 128 + t;
        if (!wait_bar(&s_full[gb & 1], (uint32_t)((gb >> 1) & 1), g, 61, gb)) ok = false;
        tc_fence_after();
        uint32_t sv[RR];
        ld_cols<RR>(tS + lane_off + NR * (gb & 1), sv);
        tmem_wait_ld();
        tc_fence_before();
        bar_arrive(&s_empty[gb & 1]);
        float x[RR];
        bool up = false;
#pragma unroll
        for (int r = 0; r < RR; ++r) {
          x[r] = key <= last_key[r] ? __uint_as_float(sv[r]) * sl : NEG_INF;
          up |= x[r] > m_ref[r] + kLazy;
        }
        if (vote_any(up)) {
          // A row's reference moves: the block's row maxima, within the warps and across them.
#pragma unroll
          for (int r = 0; r < RR; ++r) {
            float v = x[r];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
            if (lane == 0) sRed[warp * NR + r] = v;
          }
          named_barrier_sync(1, 128);
          bool resc = false;
          float alpha[RR];
#pragma unroll
          for (int r = 0; r < RR; ++r) {
            const float bm = fmaxf(fmaxf(sRed[r], sRed[NR + r]), fmaxf(sRed[2 * NR + r], sRed[3 * NR + r]));
            alpha[r] = 1.f;
            if (bm > m_ref[r] + kLazy) {
              if (m_ref[r] != NEG_INF) {
                alpha[r] = fast_exp2(m_ref[r] - bm);
                resc = true;
              }
              m_ref[r] = bm;
            }
            l_part[r] *= alpha[r];
          }
          if (resc && j > 0) {
            // Oᵀ holds PV up to block j-1: let it finish, then rescale its columns.
            if (!wait_bar(&p_empty[(gb - 1) & 1], (uint32_t)(((gb - 1) >> 1) & 1), g, 62, gb)) ok = false;
            tc_fence_after();
            uint32_t o[RR];
            ld_cols<RR>(tO + lane_off, o);
            tmem_wait_ld();
#pragma unroll
            for (int r = 0; r < RR; ++r) o[r] = __float_as_uint(__uint_as_float(o[r]) * alpha[r]);
            st_cols<RR>(tO + lane_off, o);
            tmem_wait_st();
          }
          named_barrier_sync(1, 128);     // sRed is read: the next block may write it
        }
        // Pᵀ of this block into buffer gb & 1 once the PV of block gb - 2 has read it.
        if (!wait_bar(&p_empty[gb & 1], (uint32_t)((gb >> 1) & 1) ^ 1, g, 63, gb)) ok = false;
        uint8_t* pb = sP + (gb & 1) * C::kP + (t >> 6) * NR * 128;
        const int kin = t & 63;            // key within the 64-key chunk
#pragma unroll
        for (int r = 0; r < RR; ++r) {
          const float mu = m_ref[r] == NEG_INF ? 0.f : m_ref[r] - kShift;
          const float pr = fast_exp2(x[r] - mu);
          l_part[r] += pr;
          // K-major, 128-byte swizzle: 16-byte unit (kin / 8) of row r moves to (kin / 8) ^ (r % 8).
          const int unit = (kin >> 3) ^ (r & 7);
          *reinterpret_cast<uint16_t*>(pb + r * 128 + unit * 16 + (kin & 7) * 2) = bits16<BF16>(pr);
        }
        fence_proxy_async_smem();
        tc_fence_before();
        bar_arrive(&p_full[gb & 1]);
      }

      // ---------------- epilogue of the item ----------------
      if (!wait_bar(o_full, (uint32_t)(it & 1), g, 64, it)) ok = false;
      tc_fence_after();
      uint32_t o[RR];
      ld_cols<RR>(tO + lane_off, o);
      tmem_wait_ld();
      tc_fence_before();
      bar_arrive(o_empty);
      // Row sums: each thread holds its keys' share.
#pragma unroll
      for (int r = 0; r < RR; ++r) {
        float v = l_part[r];
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
        if (lane == 0) sRed[warp * NR + r] = v;
      }
      const bool bad = vote_any(!ok);      // also the barrier between the sums' writes and reads
#pragma unroll
      for (int r = 0; r < RR; ++r) {
        const int pos = r / p.group;
        if (r >= p.nrows || pos >= im.qlen || bad) continue;
        const float l = (sRed[r] + sRed[NR + r]) + (sRed[2 * NR + r] + sRed[3 * NR + r]);
        const float ov = __uint_as_float(o[r]);
        const float m = m_ref[r] == NEG_INF ? NEG_INF : m_ref[r] - kShift;
        if (im.slot < 0) {
          const long long tok = im.tok0 + pos;
          const int h = im.hk * p.group + r - pos * p.group;
          const float inv = l == 0.f ? 0.f : 1.f / l;
          uint16_t* dst = reinterpret_cast<uint16_t*>(p.O) + tok * p.o_st + h * p.o_sh;
          if (t < D) dst[t] = bits16<BF16>(ov * inv);
          if (p.lse && t == 0)
            p.lse[tok * p.Hq + h] = l == 0.f ? NEG_INF : (m + log2f(l)) * 0.69314718055994530942f;
        } else {
          const long long at = (long long)im.slot * NR + r;
          if (t < D) p.part_o[at * D + t] = ov;
          if (t == 0) {
            p.part_ml[at * 2] = m;
            p.part_ml[at * 2 + 1] = l;
          }
        }
      }
      if (bad) break;
      named_barrier_sync(1, 128);     // the sums are read: the next item may write the slots
    }
  }

  tc_fence_before();
  __syncthreads();
  griddep_launch_dependents();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

template <int D, int NR, int RR, bool BF16>
int launch(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const DecParams& p,
           int ctas, cudaStream_t stream) {
  auto kern = paged_decode_kernel<D, NR, RR, BF16>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       Cfg<D, NR>::kSmem);
  if (e != cudaSuccess) return fail_cuda(e, "lvb_attention_paged", "cudaFuncSetAttribute (decode)");
  kern<<<ctas, kThreads, Cfg<D, NR>::kSmem, stream>>>(tq, tk, tv, p);
  e = cudaGetLastError();
  return e == cudaSuccess ? LVB_OK : fail_cuda(e, "lvb_attention_paged", "decode launch");
}

template <int D, bool BF16>
int launch_rows(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                const DecParams& p, int ctas, cudaStream_t stream) {
  if (p.nrows == 1) return launch<D, 16, 1, BF16>(tq, tk, tv, p, ctas, stream);
  if (p.nrows <= 4) return launch<D, 16, 4, BF16>(tq, tk, tv, p, ctas, stream);
  if (p.nrows <= 8) return launch<D, 16, 8, BF16>(tq, tk, tv, p, ctas, stream);
  if (p.nrows <= 16) return launch<D, 16, 16, BF16>(tq, tk, tv, p, ctas, stream);
  return launch<D, 32, 32, BF16>(tq, tk, tv, p, ctas, stream);
}

int product_rows(const lvb_paged_desc* d) {
  return (d->heads_q / d->heads_kv) * d->max_q <= 16 ? 16 : 32;
}

// One CTA per SM; fewer when even full tables would not give every CTA a block.
int decode_ctas(const lvb_paged_desc* d, int sm_count) {
  const int64_t most = (d->table_width * d->page_size + 127) / 128;
  const int64_t blocks = std::max<int64_t>(1, d->batch * d->heads_kv * std::max<int64_t>(1, most));
  return (int)std::min<int64_t>(blocks, std::max(1, sm_count));
}

size_t decode_slots(const lvb_paged_desc* d, int sm_count, bool keep_parts) {
  return 2 * (size_t)decode_ctas(d, sm_count) + (keep_parts ? (size_t)(d->batch * d->heads_kv) : 0);
}

}  // namespace

size_t paged_decode_workspace(const lvb_paged_desc* d, int sm_count, bool keep_parts) {
  return (size_t)(d->batch * d->heads_kv) * sizeof(int4) +
         decode_slots(d, sm_count, keep_parts) * product_rows(d) * (d->head_dim + 2) * sizeof(float);
}

int paged_decode_launch(const lvb_paged_desc* d, const PagedLayout& lay, const PagedSeqs& seqs,
                        const void* Q, const void* Kc, const void* Vc, void* O, float* lse,
                        bool keep_parts, void* ws, DecodeWorkspace* out, cudaStream_t stream,
                        DeviceState* dev) {
  const char* op = "lvb_attention_paged";
  DecParams p = {};
  p.seqs = seqs;
  p.Hq = (int)d->heads_q;
  p.Hkv = (int)d->heads_kv;
  p.group = p.Hq / p.Hkv;
  p.nrows = p.group * (int)d->max_q;
  p.causal = d->causal ? 1 : 0;
  p.box = paged_box(d->page_size);
  p.keep_parts = keep_parts ? 1 : 0;
  p.scale_log2 = d->scale * 1.4426950408889634f;
  p.O = O;
  p.o_st = lay.o[0];
  p.o_sh = lay.o[1];
  p.lse = lse;
  p.timeout_ns = wait_timeout_ns();
  const int rows = product_rows(d);
  const size_t slots = decode_slots(d, dev->sm_count, keep_parts);
  p.tab = reinterpret_cast<int4*>(ws);
  p.part_o = reinterpret_cast<float*>(p.tab + d->batch * d->heads_kv);
  p.part_ml = p.part_o + slots * rows * d->head_dim;
  const int ctas = decode_ctas(d, dev->sm_count);
  *out = DecodeWorkspace{p.part_o, p.part_ml, p.tab, rows, (int)slots, ctas};
  CUtensorMap tq, tk, tv;
  {
    const uint64_t dims[3] = {(uint64_t)d->head_dim, (uint64_t)d->heads_q, (uint64_t)d->tokens};
    const uint64_t str[2] = {(uint64_t)lay.q[1], (uint64_t)lay.q[0]};
    const uint32_t box[3] = {64, (uint32_t)p.group, (uint32_t)d->max_q};
    int st = make_tmap_nd(&tq, Q, 2, 3, dims, str, box, op);
    if (st) return st;
  }
  int st = paged_kv_maps(&tk, &tv, d, lay, Kc, Vc, op);
  if (st) return st;
  if (d->head_dim == 128)
    return d->dtype == LVB_BF16 ? launch_rows<128, true>(tq, tk, tv, p, ctas, stream)
                                : launch_rows<128, false>(tq, tk, tv, p, ctas, stream);
  return d->dtype == LVB_BF16 ? launch_rows<64, true>(tq, tk, tv, p, ctas, stream)
                              : launch_rows<64, false>(tq, tk, tv, p, ctas, stream);
}

}  // namespace lvb
