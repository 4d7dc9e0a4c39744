// attn_paged_decode_sm100.cu — attention of few query rows per KV head (group·max_q <= 16) over
// the paged KV cache, B200 (sm_100a).
//
// O = softmax(scale·Q·Kᵀ + mask)·V with one pass over the keys: S of a 128-key block, a running
// reference maximum m per row, p = 2^(s·log2e - m), O += P·V, l += Σp. The cache is read once at
// HBM speed, and the products are turned so that the keys fill the tensor core's 128 rows:
//   Sᵀ (128 keys × kRows) = K_j·Qᵀ,   Oᵀ (D × kRows) += V_jᵀ·P_jᵀ,   kRows = 16
// (rows = position·group + head of the group). P is rounded to the cache's type for the second
// product (the tensor core takes both operands in one 16-bit type); l sums the unrounded p.
//
//   * the 128-key blocks of all (sequence, KV head) items, one after the other, are dealt to the
//     CTAs in equal contiguous runs (an item also counts some blocks for its start and end), so
//     lengths from one key to the whole cache load the SMs evenly. The lengths are on the device:
//     every CTA sums the block counts itself. An item that a run boundary cuts leaves pieces (O, m,
//     l in 32 bits) in the workspace, at most two per CTA, and the join kernel adds them in a
//     fixed order; an item inside a run stores its result;
//   * items of at most eight blocks are not cut (paged_decode_whole): one launch, no join;
//   * with few items, or short ones (the rule is at paged_decode_cluster), an item's blocks are split
//     over a cluster of CTAs instead, which join their O, m and l through distributed shared memory:
//     one launch, no workspace, no sums over the batch (a single sequence of 777 keys 9.3 us, 11.6
//     with the join kernel). In these two forms an item's blocks may begin with a prefix's, which all
//     items share (4 sequences behind 500 keys 11.3 us, 21.0 with the prefix in a pass of its own and
//     the items dealt and joined);
//   * 384 threads: two softmax warpgroups take the blocks in turn, each with its own S and P
//     buffer, maxima, sums and O accumulator (thread = key for Sᵀ, = head-dim element for Oᵀ), so
//     one's chain of waits runs beside the other's; the one with an item's last block joins the
//     other's O (read from TMEM), m and l to its own. One warp works out
//     the items, publishes them and brings Q and the K blocks, one brings the V blocks (a box of
//     slots per page and lane), through rings that run ahead across items; one warp issues the
//     Q·Kᵀ products, one the P·V products;
//   * m of a row moves only when a score exceeds it by 2^8 (p stays <= 256): a block whose scores
//     all stay below needs no row maximum, only one vote over the warpgroup. In fp16 the exponent
//     is shifted by 2^6, away from the subnormals (p <= 2^14).
#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "paged.cuh"

namespace lvb {

namespace {

constexpr int kThreads = 384;
// Warps 0-3 and 4-7: the softmax warpgroups.
constexpr int kTmaWarp = 8;                // the items, Q and the K blocks
constexpr int kVWarp = 9;                  // the V blocks
constexpr int kQkWarp = 10;
constexpr int kPvWarp = 11;
constexpr int kRows = 16;                  // rows of the products
constexpr int kQueue = 8;                  // items published ahead
template <int D>
constexpr int kItemCost = paged_item_cost(D);   // units of an item beside its blocks
constexpr int kChunk = 128 * 128;          // one 64-element chunk of a 128-key block
constexpr float kLazy = 8.f;               // log2 units a score may exceed the reference maximum

struct DecParams {
  PagedSeqs seqs;
  int Hq, Hkv, group, nrows, causal, box, keep_parts;
  int prefix;               // keys of the prefix when every item reads it in front of its own, else 0
  int late_wait;            // 1: runs beside the kernel before it (see the kernel's start)
  int cluster;              // CTAs per item (0: the blocks of all items are dealt out)
  float scale_log2;
  void* O;
  long long o_st, o_sh;
  float* lse;
  float* part_o;            // [slot][kRows][D]
  float* part_ml;           // [slot][kRows][2]
  int4* tab;                // [batch·Hkv]; NULL: no item is cut, each goes to the CTA whose run has
                            // its first block
  unsigned long long timeout_ns;
};

template <int D>
struct Cfg {
  static constexpr int kCh = D / 64;
  static constexpr int kBlock = kCh * kChunk;
  static constexpr int kK = D == 64 ? 6 : 3;             // K ring slots
  static constexpr int kV = D == 64 ? 6 : 3;             // V ring slots
  static constexpr int kRing = kK + kV;
  static constexpr int kQ = kCh * kRows * 128;            // Q of an item
  static constexpr int kP = 2 * kRows * 128;              // P of a block: two 64-key chunks
  static constexpr int kTmemCols = 128;               // S and two O per warpgroup
  static constexpr int kSmem =
      kRing * kBlock + 2 * kQ + 2 * kP + 2 * 4 * kRows * 4 + 3 * kRows * 8 + 2048 +
      kThreads * 12 + 1024;
};

// What the roles need of an item (a run of key blocks of one sequence and KV head).
struct Item {
  int b, hk, kb0, nblk;     // sequence, KV head, first block, blocks
  int len, qlen, tok0;
  int slot;                 // where its piece goes; -1: the whole item, O is stored
  int last;                 // 1: no item, the CTA is done
  int pad;
  int entries[32];          // the table's entries from the first block's on
};

// The boxes of an item's blocks: those in the prefix, then the sequence's own.
template <int D, bool PRE>
struct ItemWalk {
  BoxWalk<D> walk;
  const int* row;
  int len, to_own;      // blocks before the sequence's own first one (0 or less: none)
  __device__ __forceinline__ void start(const BlockLane<D>& bl, const DecParams& p, const Item& im, int npb) {
    row = p.seqs.table + im.b * p.seqs.table_stride;
    len = im.len;
    to_own = npb - im.kb0;
    if (PRE && to_own > 0) walk.start(bl, p.seqs.prefix_table, im.kb0, p.prefix, p.box, p.seqs.page_size, im.entries);
    else walk.start(bl, row, -to_own, len, p.box, p.seqs.page_size, im.entries);
  }
  __device__ __forceinline__ BoxAt take(const BlockLane<D>& bl, const DecParams& p, int j) {
    if (PRE && j > 0 && j == to_own) walk.start(bl, row, 0, len, p.box, p.seqs.page_size);
    return walk.take();
  }
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
  else tmem_ld16(taddr, r);
}
template <int N>
__device__ __forceinline__ void st_cols(uint32_t taddr, uint32_t (&r)[N]) {
  if constexpr (N == 1) tmem_st1(taddr, r);
  else if constexpr (N == 4) tmem_st4(taddr, r);
  else if constexpr (N == 8) tmem_st8(taddr, r);
  else tmem_st16(taddr, r);
}

__device__ __forceinline__ void drain_wait(uint64_t* bar, uint32_t parity, uint64_t timeout_ns) {
  const uint32_t a = smem_u32(bar);
  const uint64_t t0 = global_ns();
  while (!bar_try_wait(a, parity)) {
    if (global_ns() - t0 > timeout_ns) return;
  }
}

// Whether `pred` holds for any of the warpgroup's 128 threads (named barrier `id`).
__device__ __forceinline__ bool vote_any(int id, bool pred) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %2, 0;\n\t"
      "barrier.cta.red.or.pred q, %1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"(id), "r"((uint32_t)pred)
      : "memory");
  return any != 0;
}

// A single thread's wait that tests before it suspends.
__device__ __forceinline__ bool wait_soon(uint64_t* bar, uint32_t parity, const WaitGuard& g,
                                          int where, int detail) {
  if (bar_test_wait(smem_u32(bar), parity)) return true;
  return wait_bar(bar, parity, g, where, detail);
}

// Key blocks of a sequence (0 when it has no query rows).
__device__ __forceinline__ int blocks_of(const SeqInfo& s, int npb) {
  return s.qlen > 0 ? npb + (s.len + 127) / 128 : 0;
}

// RR <= kRows: the rows that the softmax works on (the smallest of 1, 4, 8, 16 that holds the
// query rows); the products' other columns are computed and never read.
template <int D, int RR, bool BF16, bool PRE>
__global__ void __launch_bounds__(kThreads, 1)
    paged_decode_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                        const __grid_constant__ CUtensorMap tmV,
                        const __grid_constant__ DecParams p) {
  using C = Cfg<D>;
  constexpr int KR = C::kK, VR = C::kV;
  constexpr uint32_t kFmt = BF16 ? 1 : 0;
  constexpr uint32_t kIdescQK = make_idesc(1, kFmt, kFmt, 0, 0, 128, kRows);
  constexpr uint32_t kIdescPV = make_idesc(1, kFmt, kFmt, 1, 0, 128, kRows);
  constexpr float kShift = kWeightShift<BF16>;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_1024(smem_raw);
  uint8_t* sRing = smem;                                  // [KR + VR][D/64 chunks][128 keys][128 B]
  uint8_t* sQ = sRing + C::kRing * C::kBlock;                    // [2][D/64 chunks][kRows rows][128 B]
  uint8_t* sP = sQ + 2 * C::kQ;                           // [2][2 chunks][kRows rows][128 B]
  float* sXml = reinterpret_cast<float*>(sP + 2 * C::kP); // [2 warpgroups][kRows][2] deposited m, l
  float* sJml = sXml + 2 * kRows * 2;                        // [kRows][2] this CTA's part's m and l
  float* sRed = sJml + kRows * 2;                            // [2 warpgroups][4 warps][kRows]
  float* sJ = reinterpret_cast<float*>(sRing);            // [kRows][D] its O, when the ring is done with
  uint64_t* bars = reinterpret_cast<uint64_t*>(sRed + 2 * 4 * kRows);
  uint64_t* k_full = bars;               // [KR]
  uint64_t* k_empty = k_full + KR;       // [KR]
  uint64_t* v_full = k_empty + KR;       // [VR]
  uint64_t* v_empty = v_full + VR;       // [VR]
  uint64_t* q_full = v_empty + VR;       // [2]
  uint64_t* q_empty = q_full + 2;        // [2]
  uint64_t* s_full = q_empty + 2;        // [2] per warpgroup, as all below
  uint64_t* s_empty = s_full + 2;        // [2] (4 warps)
  uint64_t* p_full = s_empty + 2;        // [2] (4 warps)
  uint64_t* p_empty = p_full + 2;        // [2]
  uint64_t* o_full = p_empty + 2;        // [2][2] an item's last PV done
  uint64_t* o_empty = o_full + 4;        // [2][2] its Oᵀ read (4 warps)
  uint64_t* x_full = o_empty + 4;        // [2] the warpgroup's m and l deposited (4 warps)
  uint64_t* x_empty = x_full + 2;        // [2] they are read (4 warps of the other)
  uint64_t* i_full = x_empty + 2;        // [kQueue] item published
  uint64_t* i_empty = i_full + kQueue;   // [kQueue] read by all 12 warps
  uint64_t* drain = i_empty + kQueue;
  Item* items = reinterpret_cast<Item*>(drain + 1);       // [kQueue]
  int* sScan = reinterpret_cast<int*>(items + kQueue);    // [12] the warps' sums
  int* sStart = sScan + 12;                               // the run's sequence and its offset
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sStart + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  SeqInfo* sSeq = reinterpret_cast<SeqInfo*>(tmem_slot + 2);   // [kThreads]

  const uint32_t warp = warp_id();
  const uint32_t lane = lane_id();
  const int G = gridDim.x;

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2 * C::kRing; ++s) bar_init(&k_full[s], 1);   // all four rings' barriers
    for (int i = 0; i < 2; ++i) {
      bar_init(&q_full[i], 1);
      bar_init(&q_empty[i], 1);
      bar_init(&s_full[i], 1);
      bar_init(&s_empty[i], 4);
      bar_init(&p_full[i], 4);
      bar_init(&p_empty[i], 1);
      bar_init(&x_full[i], 4);
      bar_init(&x_empty[i], 4);
    }
    for (int i = 0; i < 4; ++i) {
      bar_init(&o_full[i], 1);
      bar_init(&o_empty[i], 4);
    }
    for (int i = 0; i < kQueue; ++i) {
      bar_init(&i_full[i], 33);     // 32 lanes' table entries and the item itself
      bar_init(&i_empty[i], 12);
    }
    bar_init(drain, 2);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kQkWarp) {
    tmem_alloc(tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }
  if (warp == kTmaWarp && lane == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }

  // The setup above may run while the stream's previous kernel ends; the join kernel, which reads
  // this one's results after its own wait, may be scheduled from here on. When the kernel before
  // this one is the same call's over the prefix, the two share only inputs, which that kernel has
  // waited for: this one then takes the SMs as they become free and waits at its end, so that its
  // own end is that kernel's too.
  if (!p.late_wait) griddep_wait();
  griddep_launch_dependents();

  const int npb = PRE ? (p.prefix + 127) / 128 : 0;    // an item's blocks: the prefix's, then its own

  // A cluster's item is given by its number: the producer reads its sequence at once.
  const int c_id = p.cluster ? blockIdx.x / p.cluster : 0, c_b = c_id / p.Hkv;
  SeqInfo c_seq{0, 0, 0};
  if (p.cluster && warp == kTmaWarp) {
    c_seq = seq_info(p.seqs, c_b);
    if (lane == 0) {
      sStart[0] = c_seq.tok0;      // for the join
      sStart[1] = c_seq.qlen;
    }
  }

  // ---------------- this CTA's run of blocks ----------------
  // Thread i sums the costs of sequences [i·per, (i+1)·per); a scan over the threads gives the
  // total and the thread whose sequences hold the run's first unit. An item's units are its
  // kItemCost<D>, then its blocks.
  const int batch = p.seqs.batch;
  const int per = (batch + kThreads - 1) / kThreads;
  const int sb0 = min((int)threadIdx.x * per, batch), sb1 = min(sb0 + per, batch);
  auto units_of = [&](int nb) -> int { return nb ? (nb + kItemCost<D>) * p.Hkv : 0; };
  const bool kept = batch <= kThreads;     // one sequence per thread: the producer reads them here
  int mine = 0;
  for (int b = p.cluster ? sb1 : sb0; b < sb1; ++b) {
    const SeqInfo s = seq_info(p.seqs, b);
    if (kept) sSeq[b] = s;
    mine += units_of(blocks_of(s, npb));
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if ((int)lane >= o) incl += v;
  }
  if (lane == 31) sScan[warp] = incl;
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < (int)warp) before += sScan[w];
    total += sScan[w];
  }
  const int share = max(1, (total + G - 1) / G);
  const int u0 = min((int)blockIdx.x, total / share + 1) * share;   // (no product above 2·total + share)
  const int u1 = min(u0 + share, total);
  const int first = before + incl - mine;
  if (p.cluster && threadIdx.x < kRows) {
    sJml[2 * threadIdx.x] = 0.f;
    sJml[2 * threadIdx.x + 1] = 0.f;       // no part yet
  }
  if (u0 < total && u0 >= first && u0 < first + mine) {
    int off = first;
    for (int b = sb0; b < sb1; ++b) {
      const int n = kept ? mine : units_of(blocks_of(seq_info(p.seqs, b), npb));
      if (u0 < off + n) {
        sStart[0] = off;
        sStart[1] = b;
        break;
      }
      off += n;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // columns: S of warpgroup w at w·kRows, its O buffers at (2 + 2w + ob)·kRows
  const WaitGuard g{p.seqs.status, abort_flag, p.timeout_ns};

  auto load_q = [&](int qb, int hk, int tok0) {
    bar_arrive_expect_tx(&q_full[qb], C::kCh * p.nrows * 128);
    for (int c = 0; c < C::kCh; ++c)
      tma_load_3d(sQ + qb * C::kQ + c * kRows * 128, &tmQ, c * 64, hk * p.group, tok0, &q_full[qb]);
  };

  if (warp == kTmaWarp) {
    // ---------------- producer: items, Q, K and V blocks ----------------
    const BlockLane<D> bl((int)lane, p.box);
    int n = 0;        // blocks loaded
    bool ok = true;
    int base = 0;     // the lanes hold sequences base .. base+31
    SeqInfo sq{0, 0, 0};
    int nb_lane = 0;
    int off = 0;      // first unit of sequence b
    int b = 0;
    auto fetch = [&]() {
      sq = SeqInfo{0, 0, 0};
      if (base + (int)lane < batch) sq = kept ? sSeq[base + lane] : seq_info(p.seqs, base + lane);
      nb_lane = blocks_of(sq, npb);
    };
    // Copy the first 32 table entries of a run that begins with block kb0.
    auto fetch_entries = [&](Item& im, int seq, int kb0, int len) {
      const bool pre = PRE && kb0 < npb;
      const int* row = pre ? p.seqs.prefix_table : p.seqs.table + seq * p.seqs.table_stride;
      const int entry = (pre ? kb0 : kb0 - npb) * 128 / p.seqs.page_size + (int)lane;
      if (entry <= ((pre ? p.prefix : len) - 1) / p.seqs.page_size) copy_async4(&im.entries[lane], row + entry);
    };
    // Publish the next item with blocks, or the end. The table entries of its first blocks are copied
    // beside it without waiting: with several items published ahead, short sequences do not wait for
    // their page numbers one after the other.
    int u = u0;
    int pub = 0;
    bool ended = false;
    auto publish = [&]() -> bool {
      const int qi = pub % kQueue;
      if (!wait_soon_warp(&i_empty[qi], (uint32_t)((pub / kQueue) & 1) ^ 1, g, 70, pub)) return false;
      Item& im = items[qi];
      bool found = false;
      if (p.cluster && pub == 0) {
        const SeqInfo& c = c_seq;
        const int rank = blockIdx.x - c_id * p.cluster;
        const int nb = blocks_of(c, npb);
        const int kb0 = (int)((long long)nb * rank / p.cluster);
        const int kb1 = (int)((long long)nb * (rank + 1) / p.cluster);
        found = kb1 > kb0;
        if (found) {
          fetch_entries(im, c_b, kb0, c.len);
          if (lane == 0) {
            im.b = c_b;
            im.hk = c_id - c_b * p.Hkv;
            im.kb0 = kb0;
            im.nblk = kb1 - kb0;
            im.len = c.len;
            im.qlen = c.qlen;
            im.tok0 = c.tok0;
            im.slot = p.cluster == 1 ? -1 : 0;
            im.last = 0;
          }
        }
      }
      while (u < u1 && !found) {
        int nb = __shfl_sync(0xffffffffu, nb_lane, b - base);
        if (u >= off + units_of(nb)) {
          // the next sequence with blocks (u < total: there is one)
          off += units_of(nb);
          int from = b + 1 - base;
          while (true) {
            const unsigned some = from < 32 ? __ballot_sync(0xffffffffu, nb_lane > 0) >> from : 0u;
            if (some) {
              b = base + from + __ffs(some) - 1;
              break;
            }
            base += 32;
            from = 0;
            fetch();
          }
          nb = __shfl_sync(0xffffffffu, nb_lane, b - base);
        }
        const int hk = (u - off) / (nb + kItemCost<D>);
        const int o_item = off + hk * (nb + kItemCost<D>) + kItemCost<D>;   // its first block
        const int kb0 = p.tab ? max(0, u - o_item) : u <= o_item ? 0 : nb;
        const int kb1 = p.tab ? min(nb, u1 - o_item) : o_item < u1 ? nb : 0;
        u = o_item + nb;
        if (kb1 <= kb0) continue;     // the run ends within the item's own cost
        found = true;
        const int len = __shfl_sync(0xffffffffu, sq.len, b - base);
        const int qlen = __shfl_sync(0xffffffffu, sq.qlen, b - base);
        const int tok0 = __shfl_sync(0xffffffffu, sq.tok0, b - base);
        const int id = b * p.Hkv + hk;
        const int c0 = o_item / share, c1 = (o_item + nb - 1) / share;
        // an item that only this CTA works on is whole; of one that begins in an earlier CTA this
        // is the run's first piece, of the other kind its last
        int slot = -1;
        if (!p.tab) slot = -1;
        else if (c1 > c0) slot = 2 * blockIdx.x + ((int)blockIdx.x == c0 ? 1 : 0);
        else if (p.keep_parts) slot = 2 * G + id;
        fetch_entries(im, b, kb0, len);
        if (lane == 0) {
          im.b = b;
          im.hk = hk;
          im.kb0 = kb0;
          im.nblk = kb1 - kb0;
          im.len = len;
          im.qlen = qlen;
          im.tok0 = tok0;
          im.slot = slot;
          im.last = 0;
          if (p.tab && kb0 == 0)
            p.tab[id] = make_int4(slot, blockIdx.x + 1, c1, slot < 0 ? kItemDone : kItemPieces);
        }
      }
      if (!found) {
        ended = true;
        if (lane == 0) im.last = 1;
      }
      copy_async_arrive(&i_full[qi]);
      if (lane == 0) bar_arrive(&i_full[qi]);
      __syncwarp();
      ++pub;
      return true;
    };
    if (u0 < u1) {
      off = sStart[0];
      b = sStart[1];
      base = b & ~31;
      fetch();
    }
    int it = 0;
    for (; ok; ++it) {
      if (pub == it && !publish()) { ok = false; break; }
      const int qi = it % kQueue;
      if (!wait_soon_warp(&i_full[qi], (uint32_t)((it / kQueue) & 1), g, 75, it)) { ok = false; break; }
      const Item& im = items[qi];
      if (im.last) break;
      const int hk = im.hk, nblk = im.nblk, tok0 = im.tok0;
      ItemWalk<D, PRE> walk;
      walk.start(bl, p, im, npb);
      __syncwarp();
      if (lane == 0) bar_arrive(&i_empty[qi]);
      if (it > 0) {        // (the first item's Q comes from the V warp, beside the first K block)
        const int qb = it & 1;
        if (!wait_soon_warp(&q_empty[qb], (uint32_t)((it >> 1) & 1) ^ 1, g, 51, it)) { ok = false; break; }
        if (lane == 0) load_q(qb, hk, tok0);
        __syncwarp();
      }
      for (int j = 0; j < nblk; ++j, ++n) {
        const BoxAt at = walk.take(bl, p, j);
        const int s = n % KR;
        if (!wait_soon_warp(&k_empty[s], (uint32_t)((n / KR) & 1) ^ 1, g, 52, n)) { ok = false; break; }
        load_block<D>(sRing + s * C::kBlock, &tmK, bl, at, p.box, hk, &k_full[s], p.seqs);
        // publish ahead, two items for one, while their queue slots are free
        for (int k = 0; k < 2 && !ended && pub < it + kQueue; ++k) {
          const bool free = bar_test_wait(smem_u32(&i_empty[pub % kQueue]), (uint32_t)((pub / kQueue) & 1) ^ 1);
          if (!__all_sync(0xffffffffu, free)) break;
          if (!publish()) { ok = false; break; }
        }
        if (!ok) break;
      }
    }
    if (!ok && lane == 0) {
      // Let the copies in flight land before the CTA's shared memory goes away.
      for (int i = max(0, n - KR); i < n; ++i)
        drain_wait(&k_full[i % KR], (uint32_t)((i / KR) & 1), p.timeout_ns);
      for (int i = max(0, it - 2); i < it; ++i)
        drain_wait(&q_full[i & 1], (uint32_t)((i >> 1) & 1), p.timeout_ns);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
  } else if (warp == kVWarp) {
    // ---------------- producer: V blocks of the published items ----------------
    const BlockLane<D> bl((int)lane, p.box);
    uint8_t* ring = sRing + KR * C::kBlock;
    int n = 0;
    bool ok = true;
    for (int it = 0; ok; ++it) {
      const int qi = it % kQueue;
      if (!wait_soon_warp(&i_full[qi], (uint32_t)((it / kQueue) & 1), g, 74, it)) { ok = false; break; }
      const Item& im = items[qi];
      const int last = im.last, hk = im.hk, nblk = im.nblk;
      if (it == 0 && !last && lane == 0) load_q(0, hk, im.tok0);
      ItemWalk<D, PRE> walk;
      if (!last) walk.start(bl, p, im, npb);
      __syncwarp();
      if (lane == 0) bar_arrive(&i_empty[qi]);
      if (last) break;
      for (int j = 0; j < nblk; ++j, ++n) {
        const BoxAt at = walk.take(bl, p, j);
        const int s = n % VR;
        if (!wait_soon_warp(&v_empty[s], (uint32_t)((n / VR) & 1) ^ 1, g, 59, n)) { ok = false; break; }
        load_block<D>(ring + s * C::kBlock, &tmV, bl, at, p.box, hk, &v_full[s], p.seqs);
      }
    }
    if (!ok && lane == 0)
      for (int i = max(0, n - VR); i < n; ++i)
        drain_wait(&v_full[i % VR], (uint32_t)((i / VR) & 1), p.timeout_ns);
    if (!ok && lane == 0 && n > 0) drain_wait(&q_full[0], 0, p.timeout_ns);
    __syncwarp();
  } else if (warp == kQkWarp || warp == kPvWarp) {
    // ---------------- MMA issuers: the warp waits, one elected lane issues ----------------
    const uint64_t r_desc = sdesc_sw128(smem_u32(sRing), 16, 1024);        // K_j, K-major
    const uint64_t q_desc = sdesc_sw128(smem_u32(sQ), 16, 1024);
    const uint64_t p_desc = sdesc_sw128(smem_u32(sP), 16, 1024);
    // V_j, MN-major. 64-wide heads: the second 64 of the product's 128 rows read the same chunk
    // again (leading offset 0) and are never looked at.
    uint8_t* v_ring = sRing + KR * C::kBlock;
    const uint64_t v_desc = sdesc_sw128(smem_u32(v_ring), D == 128 ? kChunk : 0, 1024);
    int gb = 0;       // blocks before this item
    int wi0 = 0, wi1 = 0; // items that each warpgroup had a block of
    bool ok = true;
    for (int it = 0; ok; ++it) {
      const int qi = it % kQueue;
      if (!wait_bar_warp(&i_full[qi], (uint32_t)((it / kQueue) & 1), g, 71, it)) break;
      const int nb = items[qi].nblk, kb0 = items[qi].kb0, len = items[qi].len, last = items[qi].last;
      __syncwarp();
      if (lane == 0) bar_arrive(&i_empty[qi]);
      if (last) break;
      if (warp == kQkWarp) {
        const int qb = it & 1;
        if (!wait_soon_warp(&q_full[qb], (uint32_t)((it >> 1) & 1), g, 53, it)) break;
        for (int j = 0; j < nb; ++j) {
          const int gj = gb + j, w = gj & 1, sk = gj % KR;
          if (!wait_soon_warp(&k_full[sk], (uint32_t)((gj / KR) & 1), g, 54, gj) ||
              !wait_soon_warp(&s_empty[w], (uint32_t)((gj >> 1) & 1) ^ 1, g, 55, gj)) { ok = false; break; }
          tc_fence_after();
          if (elect_one()) {
            const uint64_t ad = r_desc + (uint64_t)((sk * C::kBlock) >> 4);
            const uint64_t bd = q_desc + (uint64_t)((qb * C::kQ) >> 4);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              mma_f16_ss(tmem + kRows * w, ad + (((kk >> 2) * kChunk + (kk & 3) * 32) >> 4),
                         bd + (((kk >> 2) * kRows * 128 + (kk & 3) * 32) >> 4), kIdescQK, kk > 0 ? 1u : 0u);
            mma_commit(&s_full[w]);
            mma_commit(&k_empty[sk]);                    // K_j read
            if (j == nb - 1) mma_commit(&q_empty[qb]);   // the item's Q read for the last time
          }
          __syncwarp();
        }
      } else {
        for (int j = 0; j < nb; ++j) {
          const int gj = gb + j, w = gj & 1, sv = gj % VR;
          const int wi = w ? wi1 : wi0;
          const int ob = wi & 1;
          if (!wait_soon_warp(&v_full[sv], (uint32_t)((gj / VR) & 1), g, 56, gj)) { ok = false; break; }
          const int kb = kb0 + j, valid = PRE && kb < npb ? p.prefix - kb * 128 : len - (kb - npb) * 128;
          if (valid < 128) zero_tail<D>(smem_u32(v_ring) + sv * C::kBlock, valid);
          // the warpgroup's O buffer is free once the epilogue of its last item but one read it
          if (j < 2 && !wait_soon_warp(&o_empty[2 * w + ob], (uint32_t)((wi >> 1) & 1) ^ 1, g, 58, gj)) { ok = false; break; }
          if (!wait_soon_warp(&p_full[w], (uint32_t)((gj >> 1) & 1), g, 57, gj)) { ok = false; break; }
          tc_fence_after();
          if (elect_one()) {
            const uint64_t ad = v_desc + (uint64_t)((sv * C::kBlock) >> 4);
            const uint64_t bd = p_desc + (uint64_t)((w * C::kP) >> 4);
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)   // 16 keys per MMA
              mma_f16_ss(tmem + kRows * (2 + 2 * w + ob), ad + ((kk * 16 * 128) >> 4),
                         bd + (((kk >> 2) * kRows * 128 + (kk & 3) * 32) >> 4), kIdescPV,
                         (j < 2 && kk == 0) ? 0u : 1u);
            mma_commit(&p_empty[w]);
            mma_commit(&v_empty[sv]);                    // V_j read
            if (j + 2 >= nb) mma_commit(&o_full[2 * w + ob]);   // its last block of the item
          }
          __syncwarp();
        }
      }
      wi0 += nb > 1 || !(gb & 1);
      wi1 += nb > 1 || (gb & 1);
      gb += nb;
    }
    if (elect_one()) mma_commit(drain);
    __syncwarp();
    drain_wait(drain, 0, p.timeout_ns);
  } else {
    // ---------------- softmax and epilogue: warpgroup w takes blocks gb with gb & 1 == w -----
    const int w = warp >> 2;
    const int t = threadIdx.x & 127;                    // key within the block / Oᵀ lane (d)
    const int wl = warp & 3;
    const uint32_t lane_off = (uint32_t)(wl * 32) << 16;
    const uint32_t tS = tmem + lane_off + kRows * w;
    const int bar_id = 1 + w;
    float* red = sRed + w * 4 * kRows;
    uint8_t* pt = sP + w * C::kP + (t >> 6) * kRows * 128 + (t & 7) * 2;   // Pᵀ: this key's column
    const float NEG_INF = -INFINITY;
    const float sl = p.scale_log2;

    // Sequences without a key: zero rows (or no part for the join).
    if (w == 1 && p.cluster < 2) {
      for (int b = blockIdx.x; b < batch; b += G) {
        const SeqInfo s = seq_info(p.seqs, b);
        if (blocks_of(s, npb) > 0) continue;
        const bool rows = s.qlen > 0;
        for (int hk = p.tab ? t : p.Hkv; hk < p.Hkv; hk += 128)
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
    }

    // r / group by a product: exact for r < 16 and group <= 16
    const uint32_t inv_group = 65536u / (uint32_t)p.group + 1u;
    auto row_pos = [&](int r) -> int { return (int)((uint32_t)r * inv_group >> 16); };
    int gb = 0;       // blocks before this item
    int wi = 0;       // this warpgroup's items before this one
    int wo = 0;       // the other's
    int xn0 = 0, xn1 = 0;   // deposits of each warpgroup before this item
    for (int it = 0;; ++it) {
      const int qi = it % kQueue;
      // A wait that gave up leaves the CTA's abort flag up; every thread sees it at its next
      // wait, and the 128 leave together after a vote.
      bool ok = wait_bar(&i_full[qi], (uint32_t)((it / kQueue) & 1), g, 72, it);
      if (vote_any(bar_id, !ok)) break;
      const int nb = items[qi].nblk, kb0 = items[qi].kb0, len = items[qi].len;
      const int qlen = items[qi].qlen, tok0 = items[qi].tok0, hk = items[qi].hk;
      const int slot = items[qi].slot, last = items[qi].last;
      __syncwarp();
      if (lane == 0) bar_arrive(&i_empty[qi]);
      if (last) break;
      const int j0 = (gb & 1) == w ? 0 : 1;             // this warpgroup's first block
      const int depositor = nb > 1 ? (gb + nb) & 1 : -1;   // the one without the last block
      const int x_before = depositor == 1 ? xn1 : xn0;
      xn0 += depositor == 0;
      xn1 += depositor == 1;
      if (j0 >= nb) {                                    // the other's only block
        gb += nb;
        ++wo;
        continue;
      }
      const int n_rows = min(p.nrows, qlen * p.group);   // rows r < n_rows are real
      // Row r = position·group + head of the group sees keys up to lim0 + position.
      const int lim0 = p.causal ? len - qlen : len - 1;
      const uint32_t tO = tmem + lane_off + kRows * (2 + 2 * w + (wi & 1));
      float m_ref[RR], l_part[RR];
#pragma unroll
      for (int r = 0; r < RR; ++r) {
        m_ref[r] = NEG_INF;
        l_part[r] = 0.f;
      }
      for (int j = j0; j < nb; j += 2) {
        const int gj = gb + j;
        const uint32_t ph = (uint32_t)((gj >> 1) & 1);
        if (!wait_soon(&s_full[w], ph, g, 61, gj)) ok = false;
        __syncwarp();
        tc_fence_after();
        uint32_t sv[RR];
        ld_cols<RR>(tS, sv);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(&s_empty[w]);
        // Masked scores. Inside a run of keys that every row sees (and with all RR rows real) there
        // is nothing to mask; the two forms are apart so that no row's code has a branch.
        float x[RR];
        bool up = false;
        // (every row sees the prefix)
        const bool pre = PRE && kb0 + j < npb;
        const int first = (pre ? kb0 + j : kb0 + j - npb) * 128, lim = pre ? p.prefix - 1 : lim0;
        const bool open = first + 127 <= lim;
        if (open && n_rows >= RR) {
#pragma unroll
          for (int r = 0; r < RR; ++r) x[r] = __uint_as_float(sv[r]) * sl;
        } else {
          // row r sees the key when its position is at least key - lim
          const int key = first + t;
          const int need = p.causal && !pre ? key - lim : (key <= lim ? 0 : INT_MAX);
#pragma unroll
          for (int r = 0; r < RR; ++r)
            x[r] = r < n_rows && row_pos(r) >= need ? __uint_as_float(sv[r]) * sl : NEG_INF;
        }
#pragma unroll
        for (int r = 0; r < RR; ++r) up |= x[r] > m_ref[r] + kLazy;
        if (vote_any(bar_id, up)) {
          // A row's reference moves: the block's row maxima, within the warps and across them.
#pragma unroll
          for (int r = 0; r < RR; ++r) {
            float v = x[r];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
            if (lane == 0) red[wl * kRows + r] = v;
          }
          named_barrier_sync(bar_id, 128);
          bool resc = false;
          float alpha[RR];
#pragma unroll
          for (int r = 0; r < RR; ++r) {
            const float bm = fmaxf(fmaxf(red[r], red[kRows + r]), fmaxf(red[2 * kRows + r], red[3 * kRows + r]));
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
          if (resc && j > j0) {
            // Oᵀ holds this warpgroup's PV up to its last block: let it finish, then rescale.
            if (!wait_soon(&p_empty[w], ph ^ 1, g, 62, gj)) ok = false;
            __syncwarp();
            tc_fence_after();
            uint32_t o[RR];
            ld_cols<RR>(tO, o);
            tmem_wait_ld();
#pragma unroll
            for (int r = 0; r < RR; ++r) o[r] = __float_as_uint(__uint_as_float(o[r]) * alpha[r]);
            st_cols<RR>(tO, o);
            tmem_wait_st();
          }
          named_barrier_sync(bar_id, 128);     // red is read: the next block may write it
        }
        // Pᵀ of this block, once the PV of this warpgroup's block before has read the buffer.
        if (!wait_soon(&p_empty[w], ph ^ 1, g, 63, gj)) ok = false;
#pragma unroll
        for (int r = 0; r < RR; ++r) {
          // (a row without a key so far: a finite reference, so that -inf gives 0 and NaN stays)
          const float pr = fast_exp2(x[r] - (fmaxf(m_ref[r], -3.0e38f) - kShift));
          l_part[r] += pr;
          // K-major, 128-byte swizzle: 16-byte unit (key / 8) of row r moves to (key / 8) ^ (r % 8).
          const int unit = ((t & 63) >> 3) ^ (r & 7);
          *reinterpret_cast<uint16_t*>(pt + r * 128 + unit * 16) = bits16<BF16>(pr);
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(&p_full[w]);
      }

      // ---------------- the item's end ----------------
      // Row sums: each thread holds its keys' share. The warps' sums meet at the vote below.
#pragma unroll
      for (int r = 0; r < RR; ++r) {
        float v = l_part[r];
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
        if (lane == 0) red[wl * kRows + r] = v;
      }
      if (depositor == w) {
        if (!wait_bar(&x_empty[w], (uint32_t)(x_before & 1) ^ 1, g, 65, it)) ok = false;
        if (vote_any(bar_id, !ok)) break;
#pragma unroll
        for (int r = 0; r < RR; ++r)
          if (t == r) {
            sXml[(w * kRows + r) * 2] = m_ref[r];
            sXml[(w * kRows + r) * 2 + 1] = (red[r] + red[kRows + r]) + (red[2 * kRows + r] + red[3 * kRows + r]);
          }
        __syncwarp();
        if (lane == 0) bar_arrive(&x_full[w]);
      } else {
        const int ww = w ^ 1;
        const bool both = depositor == ww;
        if (!wait_bar(&o_full[2 * w + (wi & 1)], (uint32_t)((wi >> 1) & 1), g, 64, it)) ok = false;
        if (both && (!wait_bar(&o_full[2 * ww + (wo & 1)], (uint32_t)((wo >> 1) & 1), g, 67, it) ||
                     !wait_bar(&x_full[ww], (uint32_t)(x_before & 1), g, 66, it))) ok = false;
        if (vote_any(bar_id, !ok)) break;
        tc_fence_after();
        uint32_t o[RR];
        ld_cols<RR>(tO, o);
        tmem_wait_ld();
        float l[RR], m[RR];
#pragma unroll
        for (int r = 0; r < RR; ++r) {
          l[r] = (red[r] + red[kRows + r]) + (red[2 * kRows + r] + red[3 * kRows + r]);
          m[r] = fmaxf(m_ref[r], -3.0e38f);      // finite: 2^(m - m') is 0 or 1, not NaN
        }
        if (both) {
          // the two warpgroups' sums over the larger of their references
          uint32_t o2[RR];
          ld_cols<RR>(tmem + lane_off + kRows * (2 + 2 * ww + (wo & 1)), o2);
          tmem_wait_ld();
#pragma unroll
          for (int r = 0; r < RR; ++r) {
            const float2 x2 = *reinterpret_cast<const float2*>(&sXml[(ww * kRows + r) * 2]);
            const float m2 = fmaxf(x2.x, -3.0e38f);
            const float mm = fmaxf(m[r], m2);
            const float a1 = fast_exp2(m[r] - mm), a2 = fast_exp2(m2 - mm);
            l[r] = l[r] * a1 + x2.y * a2;
            o[r] = __float_as_uint(__uint_as_float(o[r]) * a1 + __uint_as_float(o2[r]) * a2);
            m[r] = mm;
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          bar_arrive(&o_empty[2 * w + (wi & 1)]);
          if (both) {
            bar_arrive(&o_empty[2 * ww + (wo & 1)]);
            bar_arrive(&x_empty[ww]);
          }
        }
        if (slot < 0) {
          // O = sum / l; thread r of the warpgroup stores row r's lse
          float my_l = 0.f, my_m = 0.f;
          uint16_t* base = reinterpret_cast<uint16_t*>(p.O) + tok0 * p.o_st + hk * p.group * p.o_sh + t;
#pragma unroll
          for (int r = 0; r < RR; ++r) {
            const int pos = row_pos(r), h = r - pos * p.group;
            const float inv = l[r] == 0.f ? 0.f : __frcp_rn(l[r]);
            if (r < n_rows && t < D)
              base[pos * p.o_st + h * p.o_sh] = bits16<BF16>(__uint_as_float(o[r]) * inv);
            if (t == r) my_l = l[r], my_m = m[r] - kShift;
          }
          if (p.lse && t < n_rows) {
            const int pos = row_pos(t);
            p.lse[(long long)(tok0 + pos) * p.Hq + hk * p.group + t - pos * p.group] =
                my_l == 0.f ? NEG_INF : (my_m + log2f(my_l)) * 0.69314718055994530942f;
          }
        } else if (p.cluster) {
          // The ring is read (the CTA has this one item, and its last product is done).
#pragma unroll
          for (int r = 0; r < RR; ++r) {
            if (t < D) sJ[r * D + t] = __uint_as_float(o[r]);
            if (t == r) {
              sJml[2 * r] = m[r] - kShift;
              sJml[2 * r + 1] = l[r];
            }
          }
        } else {
          const long long at = (long long)slot * kRows;
#pragma unroll
          for (int r = 0; r < RR; ++r) {
            if (r < n_rows && t < D) p.part_o[(at + r) * D + t] = __uint_as_float(o[r]);
            if (r < n_rows && t == r)
              *reinterpret_cast<float2*>(&p.part_ml[(at + r) * 2]) = make_float2(m[r] - kShift, l[r]);
          }
        }
      }
      named_barrier_sync(bar_id, 128);     // the sums are read: the next item may write them
      gb += nb;
      ++wi;
      if (nb > 1) ++wo;
    }
  }

  if (p.cluster > 1) {
    // Join the cluster's parts: row r by warp r / cluster of CTA r % cluster, D/32 elements per lane.
    // A part without a key has l = 0, and its O is not read.
    __syncthreads();
    const bool bad = *abort_flag != 0;
    if (bad && threadIdx.x < kRows) sJml[2 * threadIdx.x + 1] = -1.f;   // after a wait gave up: store nothing
    cluster_sync_all();
    const int rank = blockIdx.x - c_id * p.cluster, hk = c_id - c_b * p.Hkv;
    const int tok0 = sStart[0], n_rows = min(p.nrows, sStart[1] * p.group);
    constexpr int V = D / 32;
    const uint32_t j_addr = smem_u32(sJ) + lane * V * 4, ml_addr = smem_u32(sJml);
    for (int r = rank + (int)warp * p.cluster; r < n_rows; r += p.cluster * (kThreads / 32)) {
      float pm = -INFINITY, pl = 0.f;            // lane k: part k's m and l
      if ((int)lane < p.cluster) {
        const float2 x = ld_cluster_f32x2(mapa_shared(ml_addr + r * 8, lane));
        pm = x.x;
        pl = x.y;
      }
      // all parts' rows under way at once (of a part without a key: whatever its ring holds)
      float o[16][V];
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        if (k < p.cluster) {
          const uint32_t a = mapa_shared(j_addr + r * D * 4, k);
          if constexpr (V == 4) {
            const float4 f = ld_cluster_f32x4(a);
            o[k][0] = f.x, o[k][1] = f.y, o[k][2] = f.z, o[k][3] = f.w;
          } else {
            const float2 f = ld_cluster_f32x2(a);
            o[k][0] = f.x, o[k][1] = f.y;
          }
        }
      }
      const bool gave_up = __any_sync(0xffffffffu, pl < 0.f);
      const bool some = pl != 0.f;
      float mx = some ? pm : -INFINITY;
#pragma unroll
      for (int o2 = 16; o2 > 0; o2 >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o2));
      const float mu = mx == -INFINITY ? 0.f : mx;
      const float pw = some ? fast_exp2(pm - mu) : 0.f;
      float den = some ? pw * pl : 0.f;
#pragma unroll
      for (int o2 = 16; o2 > 0; o2 >>= 1) den += __shfl_xor_sync(0xffffffffu, den, o2);
      const unsigned parts = __ballot_sync(0xffffffffu, some);
      float acc[V];
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const float wk = __shfl_sync(0xffffffffu, pw, k);
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (parts >> k & 1) acc[e] += wk * o[k][e];
      }
      if (gave_up) continue;
      const int pos = r / p.group;
      const long long tok = tok0 + pos;
      const int h = hk * p.group + r - pos * p.group;
      const float inv = den == 0.f ? 0.f : 1.f / den;
      uint16_t* dst = reinterpret_cast<uint16_t*>(p.O) + tok * p.o_st + h * p.o_sh + lane * V;
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const uint32_t lo = bits16<BF16>(acc[e] * inv), hi = bits16<BF16>(acc[e + 1] * inv);
        *reinterpret_cast<uint32_t*>(dst + e) = lo | hi << 16;
      }
      if (p.lse && lane == 0)
        p.lse[tok * p.Hq + h] = den == 0.f ? -INFINITY : (mu + log2f(den)) * 0.69314718055994530942f;
    }
    cluster_sync_all();      // no CTA leaves while another reads its part
  }
  if (p.late_wait) griddep_wait();
  tc_fence_before();
  __syncthreads();
  if (warp == kQkWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

template <int D, int RR, bool BF16, bool PRE>
int launch(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const DecParams& p,
           int ctas, cudaStream_t stream, DeviceState* dev) {
  static SmemAttr attr;
  return launch_cluster("lvb_attention_paged", paged_decode_kernel<D, RR, BF16, PRE>, attr, dev, ctas,
                        kThreads, Cfg<D>::kSmem, std::max(1, p.cluster), stream, tq, tk, tv, p);
}

template <int D, bool BF16, bool PRE>
int launch_rows(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                const DecParams& p, int ctas, cudaStream_t stream, DeviceState* dev) {
  if (p.nrows == 1) return launch<D, 1, BF16, PRE>(tq, tk, tv, p, ctas, stream, dev);
  if (p.nrows <= 4) return launch<D, 4, BF16, PRE>(tq, tk, tv, p, ctas, stream, dev);
  if (p.nrows <= 8) return launch<D, 8, BF16, PRE>(tq, tk, tv, p, ctas, stream, dev);
  return launch<D, 16, BF16, PRE>(tq, tk, tv, p, ctas, stream, dev);
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

// As many CTAs per item as run at once, and no more than shorten the longest CTA's run. Taken when a
// full table gives a CTA at most eight blocks, so that unequal lengths cost no more than that.
int paged_decode_cluster(const lvb_paged_desc* d, const PagedRoom& room) {
  const int64_t items = d->batch * d->heads_kv;
  const int64_t blocks = std::max<int64_t>(1, (d->prefix_len + 127) / 128 + (d->table_width * d->page_size + 127) / 128);
  int c = kMostCluster;
  while (c > 0 && (c == 1 ? room.sms : room.clusters[c]) < items) --c;
  if (c == 0 || blocks > 8LL * c) return 0;
  const int64_t longest = (blocks + c - 1) / c;
  return (int)((blocks + longest - 1) / longest);
}

// Many items of at most eight blocks are dealt whole: a run's last one lengthens it by less than the
// join kernel takes. 152 items of 2, 4 and 8 blocks 12.9, 17.2 and 23.8 us, cut and joined 15.8, 18.2
// and 23.7 (the worst number of items: four CTAs have two); 400 items 18.3, 24.3 and 37.8 against 22.8,
// 28.8 and 43.9. Behind a prefix, which every item then reads again, up to 16 blocks per SM: 32 and 64
// sequences of 8 heads behind 200 keys 16.4 and 27.2 against 23.7 and 31.1 with the prefix in a pass of
// its own, behind 500 18.7 and (20 blocks per SM) 34.8 against 25.0 and 33.2.
bool paged_decode_whole(const lvb_paged_desc* d, int sm_count) {
  const int64_t blocks = (d->prefix_len + 127) / 128 + (d->table_width * d->page_size + 127) / 128;
  return blocks <= 8 && (d->prefix_len == 0 || blocks * d->batch * d->heads_kv <= 16LL * sm_count);
}

size_t paged_decode_workspace(const lvb_paged_desc* d, int sm_count, bool keep_parts) {
  return (size_t)(d->batch * d->heads_kv) * sizeof(int4) +
         decode_slots(d, sm_count, keep_parts) * kRows * (d->head_dim + 2) * sizeof(float);
}

int paged_decode_launch(const lvb_paged_desc* d, const PagedLayout& lay, const PagedSeqs& seqs,
                        const void* Q, const void* Kc, const void* Vc, void* O, float* lse,
                        bool keep_parts, bool after_prefix, int cluster, void* ws,
                        DecodeWorkspace* out, cudaStream_t stream, DeviceState* dev) {
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
  p.late_wait = after_prefix ? 1 : 0;
  p.prefix = after_prefix ? 0 : (int)d->prefix_len;
  p.cluster = cluster;
  p.scale_log2 = d->scale * 1.4426950408889634f;
  p.O = O;
  p.o_st = lay.o[0];
  p.o_sh = lay.o[1];
  p.lse = lse;
  p.timeout_ns = wait_timeout_ns();
  int ctas = cluster ? (int)(d->batch * d->heads_kv) * cluster : decode_ctas(d, dev->sm_count);
  if (ws) {
    const size_t slots = decode_slots(d, dev->sm_count, keep_parts);
    p.tab = reinterpret_cast<int4*>(ws);
    p.part_o = reinterpret_cast<float*>(p.tab + d->batch * d->heads_kv);
    p.part_ml = p.part_o + slots * kRows * d->head_dim;
    *out = DecodeWorkspace{p.part_o, p.part_ml, p.tab, kRows, (int)slots, ctas};
  }
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
  // (a form of its own: the blocks' two runs cost drafts without a prefix 35.1 us against 32.1)
  auto go = [&](auto pre) {
    constexpr bool PRE = decltype(pre)::value;
    if (d->head_dim == 128)
      return d->dtype == LVB_BF16 ? launch_rows<128, true, PRE>(tq, tk, tv, p, ctas, stream, dev)
                                  : launch_rows<128, false, PRE>(tq, tk, tv, p, ctas, stream, dev);
    return d->dtype == LVB_BF16 ? launch_rows<64, true, PRE>(tq, tk, tv, p, ctas, stream, dev)
                                : launch_rows<64, false, PRE>(tq, tk, tv, p, ctas, stream, dev);
  };
  return p.prefix > 0 ? go(std::true_type{}) : go(std::false_type{});
}

}  // namespace lvb
