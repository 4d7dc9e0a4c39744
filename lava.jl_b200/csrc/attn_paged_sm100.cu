// attn_paged_sm100.cu — flash attention of packed query rows over the paged KV cache, B200
// (sm_100a): chunks of prompts and drafts with more rows than the decoding kernel takes, and the
// part of a batch's attention that reads a shared prefix, once for the rows of all sequences.
// Also the kernel that joins the parts of a row's result.
//
// The mathematics and the inner loop are those of the dense flash kernel (attn_sm100.cu): S =
// Q·Kᵀ per 128-key block into TMEM, softmax with thread = query row (running maximum, moved only
// when it grows by more than 2^8, and sum in 32 bits), P in TMEM as the A operand of P·V, rounded
// there to the inputs' type (the tensor core takes both operands in one 16-bit type). What differs:
//   * in fp16 P is held 2^6 above its value (kWeightShift);
//   * a tile's 128 rows are (position, head of the group): all query heads of a KV head stand in
//     one tile, ppt = floor(128 / group) positions each, so a KV head's keys are read once for the
//     group, and for a shared prefix once for the tokens of all sequences;
//   * K and V blocks are gathered from their pages by the TMA warp, a box of slots per lane;
//   * an item = (sequence, KV head, pair of tiles, key range) is worked out from the lengths on
//     the device by the TMA warp, which publishes all of it through the item queue;
//   * with few items (a small chunk over a long cache, a prefix) the key blocks of a tile pair
//     are split over several CTAs, which join their O, m and l (in 32 bits) in a cluster through
//     distributed shared memory, or leave them in memory for the join kernel (the rule is at
//     paged_flash_split).
#include <algorithm>
#include <climits>
#include <cmath>

#include "paged.cuh"

namespace lvb {

namespace {

constexpr int kThreads = 352;
// Warp roles: the two MMA issuers, the TMA producer; warps 2-9 are the softmax warpgroups.
constexpr int kQkWarp = 0, kPvWarp = 1, kTmaWarp = 10;
constexpr int kChunk = 128 * 128;       // bytes of one 128-row x 64-element swizzled chunk
constexpr int kQueue = 4;

struct FlashParams {
  PagedSeqs seqs;
  int Hq, Hkv, group, ppt, causal, box;
  int own;                     // 1: the sequences' own keys are read
  int prefix;                  // prefix_len when the prefix's keys are read, else 0
  int all_rows;                // 1: one run of rows, tokens 0..tokens-1 (prefix only)
  int splits, pairs_per_seq;   // pairs_per_seq: rows of the parts' index per sequence
  int store_parts;
  int cluster;                 // CTAs per cluster (of a pair's splits), one item per CTA; 0: none
  int late_wait;               // 1: runs beside the kernel before it (see the kernel's start)
  int* counter;                // items are taken from it; NULL: item blockIdx.x, + gridDim.x, ...
  float scale_log2;
  void* O;
  long long o_st, o_sh;
  float* lse;
  float* tile_o;
  float* tile_ml;
  unsigned long long timeout_ns;
};

template <int D>
struct Cfg {
  static constexpr int kTileBytes = 128 * D * 2;  // Q tile or K/V block
  static constexpr int kQBytes = 2 * kTileBytes;
  static constexpr int kRing = D == 128 ? 5 : 8;
  static constexpr int kSmem = kQBytes + kRing * kTileBytes + 1024 + 1024;   // + barriers, queue
};

// One work item. Blocks are numbered over the prefix's (npb of them), then the sequence's own;
// the item takes blocks kb0 .. kb0 + n_blocks - 1, tile t the first n_tile[t] of them.
struct Item {
  int tok0, qlen, len, pos0, hk;
  int kb0, n_blocks, n_tile0, n_tile1;
  int part;                    // index of its 256 rows among the parts
  int last;
};

__device__ __forceinline__ void drain_wait(uint64_t* bar, uint32_t parity, uint64_t timeout_ns) {
  const uint32_t a = smem_u32(bar);
  const uint64_t t0 = global_ns();
  while (!bar_try_wait(a, parity)) {
    if (global_ns() - t0 > timeout_ns) return;
  }
}

// Ring order of an item's K/V blocks: K_0, K_1, V_0, K_2, V_1, ..., V_{nb-1}: the order in which
// the products release them.
__device__ __forceinline__ int ring_k(int j) { return j == 0 ? 0 : 2 * j - 1; }
__device__ __forceinline__ int ring_v(int j, int nb) { return j + 1 < nb ? 2 * j + 2 : 2 * j + 1; }

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (BF16) {
    __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
  } else {
    __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
  }
}

// Key blocks of a row run that ends before position `pos1` of a sequence: the prefix's, then the
// own ones up to the last row's last key.
__device__ __forceinline__ int blocks_upto(const FlashParams& p, int npb, int len, int qlen,
                                           int pos1) {
  if (!p.own) return npb;
  const int keys = p.causal ? max(0, min(len, len - qlen + pos1)) : len;
  return npb + (keys + 127) / 128;
}

// Valid keys of block kb (of the item's numbering), 128 inside a run of keys.
__device__ __forceinline__ int block_keys(const FlashParams& p, int npb, int len, int kb) {
  return min(128, kb < npb ? p.prefix - kb * 128 : len - (kb - npb) * 128);
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
    paged_flash_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                       const __grid_constant__ CUtensorMap tmV, const FlashParams p) {
  using C = Cfg<D>;
  constexpr int R = C::kRing;
  constexpr int kCh = D / 64;
  constexpr uint32_t kFmt = BF16 ? 1 : 0;
  constexpr uint32_t kIdescQK = make_idesc(1, kFmt, kFmt, 0, 0, 128, 128);
  constexpr uint32_t kIdescPV = make_idesc(1, kFmt, kFmt, 0, 1, 128, D);
  constexpr float kShift = kWeightShift<BF16>;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_1024(smem_raw);
  uint8_t* sQ = smem;                                   // [2][D/64 chunks][128 rows][128 B]
  uint8_t* sRing = sQ + C::kQBytes;                     // [R][D/64 chunks][128 rows][128 B]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sRing + R * C::kTileBytes);
  uint64_t* q_full = bars;
  uint64_t* q_empty = q_full + 1;          // the item's last QK read Q
  uint64_t* ring_full = q_empty + 1;       // [R]
  uint64_t* ring_empty = ring_full + R;    // [R]
  uint64_t* s_full = ring_empty + R;       // [2] QK_t done: the S buffer holds tile t's S
  uint64_t* s_free = s_full + 2;           // the S buffer's owner copied it out (4 warps)
  uint64_t* p_full = s_free + 1;           // [2] softmax_t wrote P_t (4 warps)
  uint64_t* pv_done = p_full + 2;          // [2] PV_t done
  uint64_t* i_full = pv_done + 2;          // [kQueue] item published
  uint64_t* i_empty = i_full + kQueue;     // [kQueue] read by 2 MMA warps, 8 softmax warps
  uint64_t* drain = i_empty + kQueue;
  Item* items = reinterpret_cast<Item*>(drain + 1);   // [kQueue]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(items + kQueue);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  // qk_after[t]: Q·Kᵀ products issued right after a copy-out of tile t's S (the P·V warp
  // lets those go first).
  volatile int* qk_after = reinterpret_cast<volatile int*>(tmem_slot + 2);   // [2]

  const uint32_t warp = warp_id();
  const uint32_t lane = lane_id();

  if (threadIdx.x == 0) {
    bar_init(q_full, 1);
    bar_init(q_empty, 1);
    for (int s = 0; s < R; ++s) {
      bar_init(&ring_full[s], 1);
      bar_init(&ring_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      bar_init(&s_full[t], 1);
      bar_init(&p_full[t], 4);
      bar_init(&pv_done[t], 1);
    }
    bar_init(s_free, 4);
    for (int s = 0; s < kQueue; ++s) {
      bar_init(&i_full[s], 1);
      bar_init(&i_empty[s], 10);
    }
    bar_init(drain, 2);
    *abort_flag = 0;
    qk_after[0] = 0;
    qk_after[1] = 0;
    fence_barrier_init();
  }
  if (warp == kQkWarp) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const WaitGuard g{p.seqs.status, abort_flag, p.timeout_ns};
  // (only into L2, so what the list holds in the end is what is read)
  if (p.prefix && warp == kTmaWarp)
    for (int i = lane * 32; i < (p.prefix + p.seqs.page_size - 1) / p.seqs.page_size; i += 32 * 32)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(p.seqs.prefix_table + i));
  // The setup above may run while the stream's previous kernel ends; what reads this kernel's
  // results after its own wait may be scheduled from here on.
  // Behind the same call's kernel over the prefix it starts at once: that one has waited for the
  // stream's earlier work before it let this one start, and shares nothing with it but inputs and
  // disjoint workspace; it waits before it ends, so that its end is also that kernel's.
  if (!p.late_wait) griddep_wait();
  griddep_launch_dependents();
  const int npb = (p.prefix + 127) / 128;
  float part_m = -INFINITY, part_l = 0.f;      // a softmax thread's row of its CTA's part (clusters)
  int part_nt = 0;

  auto load_q = [&](const Item& im) {
    bar_arrive_expect_tx(q_full, (uint32_t)(2 * kCh * p.ppt * p.group * 128));
    for (int t = 0; t < 2; ++t)
      for (int c = 0; c < kCh; ++c)
        tma_load_3d(sQ + t * C::kTileBytes + c * kChunk, &tmQ, c * 64, im.hk * p.group,
                    im.tok0 + im.pos0 + t * p.ppt, q_full);
  };

  if (warp == kTmaWarp) {
    // ---------------- scheduler + TMA producer (the whole warp) ----------------
    if (lane == 0) {
      tma_prefetch_desc(&tmQ);
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
    }
    const BlockLane<D> bl((int)lane, p.box);
    const int runs = p.all_rows ? 1 : p.seqs.batch;   // runs of rows: sequences
    const int rows2 = 2 * p.ppt;                      // positions per tile pair
    int rn = 0;          // ring slots issued
    int qi = 0;          // Q tiles issued
    bool ok = true;
    int base = 0;        // the lanes hold runs base .. base+31 ...
    int done = 0;        // ... whose first item has this number
    SeqInfo sq{0, 0, 0};
    int run = 0;         // the lane's run: the 32 stand in order of falling length, so that the
                         // items taken last, when the CTAs finish, are short ones
    int incl = 0;        // items of the lanes' runs up to and with this lane's
    auto fetch = [&]() {
      run = base + (int)lane;
      sq = SeqInfo{0, 0, 0};
      if (p.all_rows) {
        if (base + (int)lane == 0) sq.qlen = p.seqs.tokens;
      } else if (base + (int)lane < runs) {
        sq = seq_info(p.seqs, base + lane);
      }
      if (runs > 1) {
        const int key = sq.qlen > 0 ? sq.len : -1;
        int rank = 0, from = 0;
#pragma unroll 4
        for (int o = 0; o < 32; ++o) {
          const int other = __shfl_sync(0xffffffffu, key, o);
          rank += other > key || (other == key && o < (int)lane);
        }
#pragma unroll 4
        for (int o = 0; o < 32; ++o)
          if (__shfl_sync(0xffffffffu, rank, o) == (int)lane) from = o;
        run = __shfl_sync(0xffffffffu, run, from);
        sq.tok0 = __shfl_sync(0xffffffffu, sq.tok0, from);
        sq.qlen = __shfl_sync(0xffffffffu, sq.qlen, from);
        sq.len = __shfl_sync(0xffffffffu, sq.len, from);
      }
      incl = (sq.qlen + rows2 - 1) / rows2 * p.Hkv * p.splits;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if ((int)lane >= o) incl += v;
      }
    };
    fetch();
    int item = blockIdx.x;
    for (int k = 0; ok; ++k) {
      if (p.cluster && k > 0) {
        item = INT_MAX;            // the one item of this CTA is done
      } else if (p.counter) {
        if (lane == 0) item = atomicAdd(p.counter, 1);
        item = __shfl_sync(0xffffffffu, item, 0);
      } else if (k > 0) {
        item += gridDim.x;
      }
      // the run that holds it (items only grow, so the runs are passed once)
      bool end = false;
      while (item - done >= __shfl_sync(0xffffffffu, incl, 31)) {
        done += __shfl_sync(0xffffffffu, incl, 31);
        base += 32;
        if (base >= runs) {
          end = true;
          break;
        }
        fetch();
      }
      const int slot = k % kQueue;
      if (!wait_bar_warp(&i_empty[slot], (uint32_t)((k / kQueue) & 1) ^ 1, g, 73, k)) { ok = false; break; }
      if (end) {
        if (lane == 0) {
          items[slot].last = 1;
          bar_arrive(&i_full[slot]);
        }
        __syncwarp();
        break;
      }
      const int src = __ffs(__ballot_sync(0xffffffffu, item - done < incl)) - 1;
      const int before = src == 0 ? 0 : __shfl_sync(0xffffffffu, incl, max(src - 1, 0));
      Item im;
      im.tok0 = __shfl_sync(0xffffffffu, sq.tok0, src);
      im.qlen = __shfl_sync(0xffffffffu, sq.qlen, src);
      im.len = __shfl_sync(0xffffffffu, sq.len, src);
      const int b = __shfl_sync(0xffffffffu, run, src);
      // Within a run the heaviest causal pairs first: pair by pair over the KV heads, whose keys stay
      // in L2, or KV head by KV head when there are more pairs than a few rounds of the CTAs.
      const int x = item - done - before;
      const int n_pairs = (im.qlen + rows2 - 1) / rows2;
      const int split = x % p.splits;
      const int y = x / p.splits;
      int pair;
      if (n_pairs <= 2 * (int)gridDim.x) {
        pair = y / p.Hkv;
        im.hk = y - pair * p.Hkv;
      } else {
        im.hk = y / n_pairs;
        pair = y - im.hk * n_pairs;
      }
      pair = n_pairs - 1 - pair;
      im.pos0 = pair * rows2;
      int n0 = blocks_upto(p, npb, im.len, im.qlen, min(im.pos0 + p.ppt, im.qlen));
      int n1 = im.pos0 + p.ppt < im.qlen
                   ? blocks_upto(p, npb, im.len, im.qlen, min(im.pos0 + rows2, im.qlen)) : 0;
      const int n = max(n0, n1);
      // (n <= 2^24 blocks, 2^23 of a prefix and as many own ones, and splits < 2^8, no more than the
      // SMs: the products fit in 32 bits without a sign)
      im.kb0 = (int)((unsigned)n * split / p.splits);
      im.n_blocks = (int)((unsigned)n * (split + 1) / p.splits) - im.kb0;
      im.n_tile0 = min(max(n0 - im.kb0, 0), im.n_blocks);
      im.n_tile1 = min(max(n1 - im.kb0, 0), im.n_blocks);
      im.part = (b * p.pairs_per_seq + pair) * p.Hkv + im.hk;
      im.part = p.cluster ? im.part * (p.splits / p.cluster) + split / p.cluster
                          : im.part * p.splits + split;
      im.last = 0;
      if (lane == 0) {
        items[slot] = im;
        bar_arrive(&i_full[slot]);            // release: the item is visible to waiters
      }
      __syncwarp();
      if (im.n_blocks == 0) continue;
      // Q of this item once the previous item's last QK has read the old one (the first item's Q
      // comes from the P·V warp, beside the first K block).
      if (qi > 0) {
        if (!wait_bar_warp(q_empty, (uint32_t)(qi & 1) ^ 1, g, 11, k)) { ok = false; break; }
        if (lane == 0) load_q(im);
        __syncwarp();
      }
      ++qi;
      const int* row = p.seqs.table + b * p.seqs.table_stride;
      // the prefix's blocks, then the sequence's own
      BoxWalk<D> walk;
      int kb_next = im.kb0;
      auto start_run = [&]() {
        if (kb_next < npb) walk.start(bl, p.seqs.prefix_table, kb_next, p.prefix, p.box, p.seqs.page_size);
        else walk.start(bl, row, kb_next - npb, im.len, p.box, p.seqs.page_size);
      };
      start_run();
      auto next_box = [&]() -> BoxAt {
        if (kb_next == npb && kb_next > im.kb0) start_run();
        ++kb_next;
        return walk.take();
      };
      // K_j is loaded one block ahead of V_{j-1}: the boxes of the last two blocks are kept, and
      // the next block's page numbers are on their way.
      BoxAt ak = next_box(), av = ak, an = ak;
      for (int i = 0; i < 2 * im.n_blocks && ok; ++i, ++rn) {
        // Item i of the ring order: K_0; odd i: K_{(i+1)/2}, or V_{nb-1} for the last;
        // even i > 0: V_{i/2 - 1}.
        const bool is_k = i == 0 || ((i & 1) && (i + 1) / 2 < im.n_blocks);
        if (is_k) {
          const int j = (i + 1) / 2;
          av = ak;
          ak = i == 0 ? ak : an;
          if (j + 1 < im.n_blocks) an = next_box();
        } else if (i & 1) {
          av = ak;          // the last V: the block of the last K
        }
        const int s = rn % R;
        if (!wait_bar_warp(&ring_empty[s], (uint32_t)((rn / R) & 1) ^ 1, g, 12, rn)) { ok = false; break; }
        load_block<D>(sRing + s * C::kTileBytes, is_k ? &tmK : &tmV, bl, is_k ? ak : av, p.box,
                      im.hk, &ring_full[s], p.seqs);
      }
    }
    if (!ok && lane == 0) {
      // Let every copy in flight land before the CTA's shared memory goes away.
      if (qi > 0) drain_wait(q_full, (uint32_t)((qi - 1) & 1), p.timeout_ns);
      for (int i = max(0, rn - R); i < rn; ++i)
        drain_wait(&ring_full[i % R], (uint32_t)((i / R) & 1), p.timeout_ns);
    }
    __syncwarp();
  } else if (warp == kQkWarp || warp == kPvWarp) {
    // ---------------- MMA issuers: one warp the Q·Kᵀ products, one the P·V products ----
    const bool qk_role = warp == kQkWarp;
    const uint32_t q_base = smem_u32(sQ);
    const uint32_t r_base = smem_u32(sRing);
    const uint64_t qd0 = sdesc_sw128(q_base, 16, 1024);
    const uint64_t kd0 = sdesc_sw128(r_base, 16, 1024);
    const uint64_t vd0 = sdesc_sw128(r_base, kChunk, 1024);
    constexpr uint32_t kTile16 = C::kTileBytes >> 4;
    int rc = 0;               // ring slots of the items before the current one
    int qi = 0;               // items with work before the current one
    int gt[2] = {0, 0};       // blocks of each tile before the current item
    int fills = 0;            // Q·Kᵀ products written to the S buffer so far
    int prev_tile = 0;        // tile of the last S written
    int after[2] = {0, 0};    // copy of qk_after (written by the Q·Kᵀ warp only)
    bool ok = true;
    for (int k = 0; ok; ++k) {
      const int islot = k % kQueue;
      if (!wait_bar_warp(&i_full[islot], (uint32_t)((k / kQueue) & 1), g, 19, k)) break;
      const Item it = items[islot];
      __syncwarp();
      if (elect_one()) bar_arrive(&i_empty[islot]);
      if (it.last) break;
      if (it.n_blocks == 0) continue;
      if (!qk_role && qi == 0 && lane == 0) load_q(it);
      __syncwarp();
      const int nt[2] = {it.n_tile0, it.n_tile1};
      const int nb = it.n_blocks;
      int ring_seen = -1;     // this warp's ring slots of the item already waited for
      auto ring_wait = [&](int i, int where) -> bool {
        if (i <= ring_seen) return true;
        const int x = rc + i;
        if (!wait_soon_warp(&ring_full[x % R], (uint32_t)((x / R) & 1), g, where, i)) return false;
        ring_seen = i;
        return true;
      };
      auto release = [&](int i) {
        if (elect_one()) mma_commit(&ring_empty[(rc + i) % R]);
        __syncwarp();
      };
      if (qk_role) {
        if (!wait_bar_warp(q_full, (uint32_t)(qi & 1), g, 12, k)) break;
        const int n_qk = nt[0] + nt[1];
        int qk_done = 0;
        auto fill = [&](int t, int j) -> bool {
          if (!ring_wait(ring_k(j), 13)) return false;
          if (fills > 0 && !wait_soon_warp(s_free, (uint32_t)((fills - 1) & 1), g, 17, j))
            return false;
          tc_fence_after();
          const bool last = ++qk_done == n_qk;
          if (elect_one()) {
            const uint64_t ad = qd0 + (uint64_t)(t * kTile16);
            const uint64_t bd = kd0 + (uint64_t)(((rc + ring_k(j)) % R) * kTile16);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const uint32_t o = ((kk >> 2) * kChunk + (kk & 3) * 32) >> 4;
              mma_f16_ss(tmem, ad + o, bd + o, kIdescQK, kk > 0 ? 1u : 0u);
            }
            mma_commit(&s_full[t]);
            if (last) mma_commit(q_empty);
          }
          __syncwarp();
          if (fills > 0) {
            ++after[prev_tile];
            if (lane == 0) qk_after[prev_tile] = after[prev_tile];
          }
          prev_tile = t;
          ++fills;
          return true;
        };
        // Fill order S_0(0), S_1(0), S_0(1), S_1(1), ... A tile may have fewer blocks than the
        // other, or none (a key range behind a causal tile's last key).
        if (nt[0] > 0) ok = fill(0, 0);
        if (ok && nt[1] > 0) ok = fill(1, 0);
        if (ok && nt[0] > 1) ok = fill(0, 1);
        if (!ok) break;
        release(0);                                              // K_0
        for (int j = 0; j < nb && ok; ++j) {
          if (j + 1 < nt[1]) ok = fill(1, j + 1);
          if (ok && j + 2 < nt[0]) ok = fill(0, j + 2);
          if (!ok) break;
          if (j + 1 < nb) release(ring_k(j + 1));                // K_{j+1}: last use
        }
      } else {
        for (int j = 0; j < nb && ok; ++j) {
          if (!ring_wait(ring_v(j, nb), 14)) { ok = false; break; }
          const int valid = block_keys(p, npb, it.len, it.kb0 + j);
          if (valid < 128)
            zero_tail<D>(r_base + ((rc + ring_v(j, nb)) % R) * C::kTileBytes, valid);
          for (int t = 0; t < 2; ++t) {
            if (j >= nt[t]) continue;
            if (!wait_soon_warp(&p_full[t], (uint32_t)((gt[t] + j) & 1), g, 15, j)) {
              ok = false;
              break;
            }
            // P_t(j) was announced with the copy-out of S_t(j+1); the Q·Kᵀ that follows it (if
            // this item has one: a softmax waits for it) goes to the tensor core before this
            // P·V. A priority hint only: after ~2 us the P·V goes anyway.
            const bool follows = j + 2 < nt[0] || (t == 0 ? j + 1 : j + 2) < nt[1];
            if (j + 1 < nt[t] && follows) {
              const int target = gt[t] + j + 2;
              if (qk_after[t] < target) {
                const uint64_t t0 = global_ns();
                while (qk_after[t] < target && global_ns() - t0 < 2000) {
                }
              }
              __syncwarp();
            }
            tc_fence_after();
            if (elect_one()) {
              const uint64_t bd = vd0 + (uint64_t)(((rc + ring_v(j, nb)) % R) * kTile16);
              const uint32_t tp = tmem + 128 + 64 * t;
#pragma unroll
              for (int kk = 0; kk < 8; ++kk)   // 128 keys, 16 per MMA: P columns 8kk..8kk+7
                mma_f16_ts(tmem + 256 + 128 * t, tp + 8 * kk, bd + (uint64_t)(kk * 128),
                           kIdescPV, (j > 0 || kk > 0) ? 1u : 0u);
              mma_commit(&pv_done[t]);
            }
            __syncwarp();
          }
          if (!ok) break;
          release(ring_v(j, nb));                                // V_j
        }
      }
      rc += 2 * nb;
      gt[0] += nt[0];
      gt[1] += nt[1];
      ++qi;
    }
    if (elect_one()) mma_commit(drain);
    __syncwarp();
    drain_wait(drain, 0, p.timeout_ns);
  } else {
    // ---------------- softmax, one warpgroup per query tile ----------------
    const int t = (warp - 2) >> 2;
    const int wl = warp & 3;
    const int r = wl * 32 + lane;               // row within the tile = TMEM lane
    const uint32_t lane_off = (uint32_t)(wl * 32) << 16;
    const uint32_t tS = tmem + lane_off;                  // the S buffer (shared)
    const uint32_t tP = tmem + lane_off + 128 + 64 * t;   // P_t
    const uint32_t tO = tmem + lane_off + 256 + 128 * t;
    const float NEG_INF = -INFINITY;
    const float sl = p.scale_log2;
    const int row_pos = r / p.group;            // position within the tile
    const int row_head = r - row_pos * p.group;
    int gt = 0;               // blocks of this tile before the current item
    bool ok = true;
    for (int k = 0; ok; ++k) {
      const int islot = k % kQueue;
      if (!wait_bar_warp(&i_full[islot], (uint32_t)((k / kQueue) & 1), g, 20, k)) break;
      const Item it = items[islot];
      __syncwarp();
      if (lane == 0) bar_arrive(&i_empty[islot]);
      if (it.last) break;
      const int pos = it.pos0 + t * p.ppt + row_pos;
      const bool row_ok = row_pos < p.ppt && pos < it.qlen;
      float m_ref = NEG_INF;   // running max (log2 domain, scale folded in)
      float l = 0.f;           // running sum of p relative to m_ref - kShift
      const int nt = t ? it.n_tile1 : it.n_tile0;
      // Keys of the sequence's own that the row sees, and that every row of the tile sees.
      const int own_keys = p.causal ? min(it.len, max(0, it.len - it.qlen + pos + 1)) : it.len;
      const int own_all = p.causal ? it.len - it.qlen + it.pos0 + t * p.ppt + 1 : it.len;

      for (int j = 0; j < nt; ++j) {
        if (!wait_bar_warp(&s_full[t], (uint32_t)((gt + j) & 1), g, 21, j)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t s[128];
        tmem_ld32(tS + 0, *reinterpret_cast<uint32_t (*)[32]>(&s[0]));
        tmem_ld32(tS + 32, *reinterpret_cast<uint32_t (*)[32]>(&s[32]));
        tmem_ld32(tS + 64, *reinterpret_cast<uint32_t (*)[32]>(&s[64]));
        tmem_ld32(tS + 96, *reinterpret_cast<uint32_t (*)[32]>(&s[96]));
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (j > 0) bar_arrive(&p_full[t]);
          bar_arrive(s_free);
        }
        const int kb = it.kb0 + j;
        // keys of this block that the row sees / that every row of the tile sees
        const bool pre = kb < npb;
        const int see = pre ? p.prefix - kb * 128 : own_keys - (kb - npb) * 128;
        const int all = pre ? see : min(own_all, it.len) - (kb - npb) * 128;
        if (all < 128) {
#pragma unroll
          for (int c = 0; c < 128; ++c)
            if (c >= see) s[c] = __float_as_uint(NEG_INF);
        }
        // Row max: 4 independent chains of 3-input maxima.
        float mxp[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) mxp[i] = __uint_as_float(s[i]);
#pragma unroll
        for (int c = 4; c < 124; c += 8)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            mxp[i] = fmax3(mxp[i], __uint_as_float(s[c + i]), __uint_as_float(s[c + 4 + i]));
#pragma unroll
        for (int i = 0; i < 4; ++i) mxp[i] = fmaxf(mxp[i], __uint_as_float(s[124 + i]));
        const float m_new = fmaxf(fmaxf(mxp[0], mxp[1]), fmaxf(mxp[2], mxp[3])) * sl;
        float alpha = 1.f;
        bool resc = false;
        if (j == 0) {
          m_ref = m_new;
        } else if (m_new > m_ref + 8.f) {
          alpha = fast_exp2(m_ref - m_new);
          m_ref = m_new;
          resc = true;
        }
        const float m_use = (m_ref == NEG_INF ? 0.f : m_ref) - kShift;
        float sump[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 64; ++c) {
          const float p0 = fast_exp2(fmaf(__uint_as_float(s[2 * c]), sl, -m_use));
          const float p1 = fast_exp2(fmaf(__uint_as_float(s[2 * c + 1]), sl, -m_use));
          sump[c & 3] += p0 + p1;
          s[c] = pack2<BF16>(p0, p1);
        }
        const float sum = (sump[0] + sump[1]) + (sump[2] + sump[3]);
        // PV_t(j-1) has finished: P_t may be rewritten and O_t rescaled.
        if (j > 0) {
          if (!wait_bar_warp(&pv_done[t], (uint32_t)((gt + j - 1) & 1), g, 22, j)) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (__any_sync(0xffffffffu, resc)) {
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t o[16];
              tmem_ld16(tO + 16 * c, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tmem_st16(tO + 16 * c, o);
            }
          }
        }
        tmem_st32(tP + 0, &s[0]);
        tmem_st32(tP + 32, &s[32]);
        tmem_wait_st();
        l = l * alpha + sum;
        tc_fence_before();
      }
      if (!ok) break;
      if (nt > 0) {
        __syncwarp();
        if (lane == 0) bar_arrive(&p_full[t]);    // the last block's P
      }

      // ---------------- epilogue: O / l -> global, lse; or the part for the join ----------------
      if (nt > 0 && !wait_bar_warp(&pv_done[t], (uint32_t)((gt + nt - 1) & 1), g, 23, 0)) break;
      tc_fence_after();
      const long long tok = it.tok0 + pos;
      const int h = it.hk * p.group + row_head;
      if (p.cluster) {
        // O stays in TMEM until the CTA's products are done (below)
        part_m = m_ref - kShift;
        part_l = l;
        part_nt = nt;
      } else if (p.store_parts) {
        const long long at = (long long)it.part * 256 + t * 128 + r;
        if (row_ok) {
          p.tile_ml[at * 2] = m_ref - kShift;
          p.tile_ml[at * 2 + 1] = l;
        }
        if (nt > 0) {
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(tO + 32 * c, o);
            tmem_wait_ld();
            if (row_ok) {
#pragma unroll
              for (int e = 0; e < 4; ++e) st_global_v8(p.tile_o + at * D + 32 * c + 8 * e, &o[8 * e]);
            }
          }
        }
        tc_fence_before();
      } else {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        uint8_t* orow = reinterpret_cast<uint8_t*>(p.O) + 2 * (tok * p.o_st + h * p.o_sh);
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          if (nt > 0) {
            tmem_ld32(tO + 32 * c, o);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0u;
          }
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; ++e)
            pk[e] = pack2<BF16>(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
          if (row_ok) {
            uint8_t* dst = orow + c * 64;
            if ((reinterpret_cast<uintptr_t>(dst) & 31) == 0) {
              // 32-byte stores: each lane's store fills a whole 32-byte sector of its row.
              st_global_v8(dst, &pk[0]);
              st_global_v8(dst + 32, &pk[8]);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                reinterpret_cast<uint4*>(dst)[e] =
                    make_uint4(pk[4 * e], pk[4 * e + 1], pk[4 * e + 2], pk[4 * e + 3]);
            }
          }
        }
        tc_fence_before();
        if (p.lse && row_ok) {
          const float mu = (m_ref == NEG_INF ? 0.f : m_ref) - kShift;
          p.lse[tok * p.Hq + h] = l == 0.f ? NEG_INF : (mu + log2f(l)) * 0.69314718055994530942f;
        }
      }
      gt += nt;
    }
  }

  if (p.cluster) {
    // The cluster's join. Each CTA copies its O, and m and l, into shared memory over Q and the ring
    // (16-byte unit c of row r at c ^ (r % 8): the threads of a store lie in different banks); row r
    // of the pair is then joined by CTA r % cluster.
    constexpr int V = D / 32;
    float* sO = reinterpret_cast<float*>(smem);               // [256][D]
    float2* sMl = reinterpret_cast<float2*>(smem + 256 * D * 4);
    tc_fence_before();
    __syncthreads();          // every product and copy of this CTA is done
    tc_fence_after();
    const bool bad = *abort_flag != 0;
    if (warp != kQkWarp && warp != kPvWarp && warp != kTmaWarp) {
      const int t = (warp - 2) >> 2, wl = warp & 3, r = t * 128 + wl * 32 + lane;
      const uint32_t tO = tmem + ((uint32_t)(wl * 32) << 16) + 256 + 128 * t;
      sMl[r] = make_float2(part_m, bad ? -1.f : part_l);      // after a wait gave up: store nothing
      if (part_nt > 0) {
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(tO + 32 * c, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 8; ++e)
            st_shared_v4(smem_u32(sO) + r * D * 4 + (((8 * c + e) ^ (r & 7)) << 4), o[4 * e],
                         o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
        }
      }
    }
    cluster_sync_all();
    const Item& im = items[0];
    const int rank = blockIdx.x % p.cluster;
    const int rows = im.last ? 0 : 256;
    const uint32_t o_addr = smem_u32(sO), ml_addr = smem_u32(sMl);
    for (int r = rank + (int)warp * p.cluster; r < rows; r += p.cluster * (kThreads / 32)) {
      const int t = r >> 7, row_pos = (r & 127) / p.group;
      const int pos = im.pos0 + t * p.ppt + row_pos;
      if (row_pos >= p.ppt || pos >= im.qlen) continue;
      float pm = -INFINITY, pl = 0.f;            // lane k: part k's m and l
      if ((int)lane < p.cluster) {
        const float2 x = ld_cluster_f32x2(mapa_shared(ml_addr + r * 8, lane));
        pm = x.x;
        pl = x.y;
      }
      // all parts' rows under way at once (of a part without a key: whatever lies there)
      const uint32_t col = V == 4 ? ((lane ^ (r & 7)) << 4) : (((lane >> 1) ^ (r & 7)) << 4) + (lane & 1) * 8;
      float o[16][V];
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        if (k < p.cluster) {
          const uint32_t a = mapa_shared(o_addr + r * D * 4 + col, k);
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
      for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      const float mu = mx == -INFINITY ? 0.f : mx;
      const float pw = some ? fast_exp2(pm - mu) : 0.f;
      float den = some ? pw * pl : 0.f;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) den += __shfl_xor_sync(0xffffffffu, den, x);
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
      if (p.store_parts) {
        // one part for the join with the sequences' own
        const long long at = (long long)im.part * 256 + r;
        if (lane == 0) *reinterpret_cast<float2*>(&p.tile_ml[at * 2]) = make_float2(mu, den);
        float* dst = p.tile_o + at * D + lane * V;
        if constexpr (V == 4) *reinterpret_cast<float4*>(dst) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        else *reinterpret_cast<float2*>(dst) = make_float2(acc[0], acc[1]);
      } else {
        const long long tok = im.tok0 + pos;
        const int h = im.hk * p.group + (r & 127) - row_pos * p.group;
        const float inv = den == 0.f ? 0.f : 1.f / den;
        uint16_t* dst = reinterpret_cast<uint16_t*>(p.O) + tok * p.o_st + h * p.o_sh + lane * V;
#pragma unroll
        for (int e = 0; e < V; e += 2)
          *reinterpret_cast<uint32_t*>(dst + e) = pack2<BF16>(acc[e] * inv, acc[e + 1] * inv);
        if (p.lse && lane == 0)
          p.lse[tok * p.Hq + h] = den == 0.f ? -INFINITY : (mu + log2f(den)) * 0.69314718055994530942f;
      }
    }
    cluster_sync_all();      // no CTA leaves while another reads its part
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kQkWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (p.late_wait) griddep_wait();
}

// ----------------------------------------------------------------------------------------
// The join: O = Σ 2^(m_s - m) O_s / Σ 2^(m_s - m) l_s, m = max m_s, over a row's parts in a fixed
// order (the prefix's or the tile's key ranges, then the decoding kernel's pieces). One, two or
// four warps per row, four parts each at a time, D/32 elements per lane. Bound by the latency of
// its loads (the lists, the item's table entry, the parts), so the parts' rows are loaded beside
// their (m, l), before their weights are known, rows of many parts take several warps, and the
// registers are kept to eight CTAs per SM: with eight parts at a time there are five, and a call over a
// prefix of 16,384 keys takes 88.1 us against 85.8, drafts over 64-wide heads 34.3 against 32.3.
// ----------------------------------------------------------------------------------------
constexpr int kMergeThreads = 128;
constexpr int kMergeParts = 4;       // parts of a row under way per warp

template <int D, bool BF16>
__global__ void __launch_bounds__(kMergeThreads, 8) merge_kernel(const MergeParams p, int rows) {
  constexpr int V = D / 32;            // elements per lane
  __shared__ float2 sh_ml[4];
  __shared__ float sh_acc[4][D];
  const int lane = lane_id();
  const int warp = warp_id();
  griddep_launch_dependents();
  // row = (sequence, position, head); a row's warps lie side by side
  const int wpr = p.warps_per_row;
  const int row = (blockIdx.x * 4 + warp) / wpr;
  const int sub = warp & (wpr - 1);
  const int bq = row / p.Hq;
  const int h = row - bq * p.Hq;
  const int b = bq / p.seqs.max_q;
  const int pos = bq - b * p.seqs.max_q;
  // The lists are older than the kernel before this one; what that kernel wrote is not. Every
  // warp waits for it, so that this grid's end is also that kernel's.
  SeqInfo s{0, 0, 0};
  if (row < rows) s = seq_info(p.seqs, b);
  bool on = pos < s.qlen;
  const long long tok = s.tok0 + pos;
  const int hk = h / p.group, gh = h - hk * p.group;
  // where the parts are
  const int nt = p.tile_splits;
  long long tile0 = 0;
  if (nt) {
    const int at = p.pairs_per_seq ? pos : (int)tok;
    const int in_pair = at % (2 * p.ppt);
    const long long pair = at / (2 * p.ppt) + (long long)b * p.pairs_per_seq;
    const int t = in_pair / p.ppt;
    tile0 = (pair * p.Hkv + hk) * nt * 256 + t * 128 + (in_pair - t * p.ppt) * p.group + gh;
  }
  long long own0 = 0;
  if (p.own_splits) {
    const int in_pair = pos % (2 * p.ppt);
    const long long pair = pos / (2 * p.ppt) + (long long)b * p.own_pairs;
    const int t = in_pair / p.ppt;
    own0 = (pair * p.Hkv + hk) * p.own_splits * 256 + t * 128 + (in_pair - t * p.ppt) * p.group + gh;
  }
  griddep_wait();
  int nd = p.own_splits, first_slot = 0, next_c = 0;
  if (p.dec_tab && on) {
    const int4 e = p.dec_tab[b * p.Hkv + hk];
    if (e.w == kItemPieces && e.x >= 0 && e.x < p.dec_slots && e.y > 0 && e.z < p.dec_ctas) {
      first_slot = e.x;
      next_c = e.y;
      nd = 1 + max(0, e.z - e.y + 1);
    } else if (e.w != kItemNoKeys || !nt) {
      on = false;                        // the decoding kernel has stored the row
    }
  }
  const int dec_row = pos * p.group + gh;
  const int n = on ? nt + nd : 0;
  // A running maximum m, and sums relative to it. A part without a key has l = 0 and an O that
  // nothing wrote: its weight is 0 and its row is dropped.
  float m = -INFINITY, den = 0.f;
  float acc[V];
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] = 0.f;
  for (int i0 = kMergeParts * sub; i0 < n; i0 += kMergeParts * wpr) {
    float v[kMergeParts][V];
    float2 ml[kMergeParts];
#pragma unroll
    for (int q = 0; q < kMergeParts; ++q) {
      const int i = min(i0 + q, n - 1), k = i - nt;
      const bool tile = k < 0;
      const long long slot = k <= 0 ? first_slot : 2 * (next_c + k - 1);
      const long long r = tile ? tile0 + (long long)i * 256
                          : p.own_splits ? own0 + (long long)k * 256 : slot * p.dec_rows + dec_row;
      ml[q] = *reinterpret_cast<const float2*>((tile ? p.tile_ml : p.own_ml) + 2 * r);
      const float* src = (tile ? p.tile_o : p.own_o) + r * D + lane * V;
      if constexpr (V == 4) {
        const float4 f = *reinterpret_cast<const float4*>(src);
        v[q][0] = f.x, v[q][1] = f.y, v[q][2] = f.z, v[q][3] = f.w;
      } else {
        const float2 f = *reinterpret_cast<const float2*>(src);
        v[q][0] = f.x, v[q][1] = f.y;
      }
    }
    float mn = m;
#pragma unroll
    for (int q = 0; q < kMergeParts; ++q) mn = fmaxf(mn, ml[q].y == 0.f ? -INFINITY : ml[q].x);
    const float mu = mn == -INFINITY ? 0.f : mn;
    const float keep = exp2f(m - mu);
    den *= keep;
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] *= keep;
#pragma unroll
    for (int q = 0; q < kMergeParts; ++q) {
      const bool in = i0 + q < n && ml[q].y != 0.f;
      const float wq = in ? exp2f(ml[q].x - mu) : 0.f;
      den += in ? wq * ml[q].y : 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] += in ? wq * v[q][e] : 0.f;
    }
    m = mn;
  }
  if (wpr > 1) {
    // the row's warps: sums relative to the largest of their maxima
    sh_ml[warp] = make_float2(m, den);
#pragma unroll
    for (int e = 0; e < V; ++e) sh_acc[warp][lane * V + e] = acc[e];
    __syncthreads();
    if (sub) return;
    float mn = m;
    for (int q = 1; q < wpr; ++q) mn = fmaxf(mn, sh_ml[warp + q].x);
    const float mu = mn == -INFINITY ? 0.f : mn;
    const float keep = exp2f(m - mu);
    den *= keep;
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] *= keep;
    for (int q = 1; q < wpr; ++q) {
      const float wq = exp2f(sh_ml[warp + q].x - mu);
      den += wq * sh_ml[warp + q].y;
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] += wq * sh_acc[warp + q][lane * V + e];
    }
    m = mn;
  }
  if (!on) return;
  const float inv = den == 0.f ? 0.f : 1.f / den;
  uint16_t* dst = reinterpret_cast<uint16_t*>(p.O) + tok * p.o_st + h * p.o_sh + lane * V;
#pragma unroll
  for (int e = 0; e < V; e += 2)
    *reinterpret_cast<uint32_t*>(dst + e) = pack2<BF16>(acc[e] * inv, acc[e + 1] * inv);
  if (p.lse && lane == 0)
    p.lse[tok * p.Hq + h] = den == 0.f ? -INFINITY : (m + log2f(den)) * 0.69314718055994530942f;
}

template <int D, bool BF16>
int launch_flash(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                 const FlashParams& p, int ctas, cudaStream_t stream, DeviceState* dev) {
  static SmemAttr attr;
  return launch_cluster("lvb_attention_paged", paged_flash_kernel<D, BF16>, attr, dev, ctas, kThreads,
                        Cfg<D>::kSmem, std::max(1, p.cluster), stream, tq, tk, tv, p);
}

constexpr size_t kCounterBytes = 256;   // the item counter, before the 32-byte stores' parts

constexpr double kBlockUs = 1.8;        // a key block of a tile pair
constexpr double kJoinUs = 4.0;         // the join kernel
constexpr double kPassUs = 16.0;        // a prefix's own pass: two more starts and ends

int positions_per_tile(const lvb_paged_desc* d) {
  return (int)(128 / (d->heads_q / d->heads_kv));
}

// Tile pairs per run of rows (all tokens for the prefix alone, max_q for a sequence).
int64_t tile_pairs(const lvb_paged_desc* d, int parts) {
  const int64_t rows = parts == kFlashPrefix ? d->tokens : d->max_q;
  const int64_t rows2 = 2 * positions_per_tile(d);
  return (rows + rows2 - 1) / rows2;
}

}  // namespace

// Items without the splits, at most.
int64_t paged_flash_items(const lvb_paged_desc* d, int parts) {
  return tile_pairs(d, parts) * d->heads_kv * (parts == kFlashPrefix ? 1 : d->batch);
}

// With fewer items than SMs: key ranges (of the prefix's length; of a table's row otherwise), by the
// cost of a CTA's blocks (1.8 us each) and of a part that goes through memory (0.45 us with its
// share of the join). With more items than half the SMs two ranges of each would not run at once,
// and an item stays whole: 9 sequences of four drafts, 64 heads on 8, over 16,384 keys are 72 items
// and take 110.9 us where their bytes take 92.4, 10 are 80 items and take 202.7 where theirs take
// 102.6. Ranges meet in clusters where that spares the join kernel or most of its work (a
// cluster's join 1.5 us, the kernel 4 us): 64 new tokens of one sequence over 1,000, 4,000 and
// 16,000 keys 14.8, 20.3 and 35.4 us with clusters, 21.6, 26.9 and 38.9 without. Parts that are
// joined anyway (a prefix's and those beside it) do not: the kernel behind it fills the SMs as the
// CTAs end (16,384 keys before 64 sequences 87.2 us with clusters, 84.9 without), and cost a tenth
// in the join, as more is going on (4,099 keys over 64-wide heads in 16 ranges 31.0 us, in 11 34.5).
FlashSplit paged_flash_split(const lvb_paged_desc* d, const PagedRoom& room, int parts, bool joined) {
  const int64_t items = std::max<int64_t>(1, paged_flash_items(d, parts));
  int64_t keys = 0;
  if (parts & kFlashPrefix) keys += d->prefix_len;
  if (parts & kFlashOwn) keys += d->table_width * d->page_size;
  const int64_t blocks = std::max<int64_t>(1, (keys + 127) / 128);
  FlashSplit best{1, 1, kBlockUs * (double)blocks * (double)((items + room.sms - 1) / room.sms)};
  if (2 * items > room.sms) return best;
  best.us = 1e30;
  for (int c = 1; c <= (joined ? 1 : kMostCluster); ++c) {
    const int64_t most = (c == 1 ? room.sms : room.clusters[c]) / items;   // groups that run at once
    for (int64_t g = 1; g <= most && g * c <= blocks; ++g) {
      const double cost = kBlockUs * (double)((blocks + g * c - 1) / (g * c)) +
                          (joined ? 0.05 : 0.45) * (double)g + (c > 1 ? 1.5 : 0.0) +
                          (!joined && g > 1 ? kJoinUs : 0.0);
      if (cost < best.us - 1e-9) best = FlashSplit{(int)(g * c), c, cost};
    }
  }
  return best;
}

size_t paged_flash_workspace(const lvb_paged_desc* d, FlashSplit fs, int parts, bool joined) {
  const int groups = fs.splits / fs.cluster;
  const bool store = joined || groups > 1;
  return kCounterBytes + (store ? (size_t)paged_flash_items(d, parts) * groups * 256 *
                                      (d->head_dim + 2) * sizeof(float) : 0);
}

// Whether the prefix is read in a pass of its own, whose tiles hold the rows of all sequences, and
// joined with the sequences' own parts, or by every sequence's tiles in front of its own keys.
// The first has fewer tiles where a sequence's rows do not fill one, but its parts go through
// memory (twice a row's D fp32, written and read) and into a join, and each pass has its start: of
// 32 sequences with 4 tokens, 64 heads on 8, and 300 own keys behind 16,384 the first takes 94.1 us,
// the second 372.8; of 16 with 8, 32 and 64 tokens, 32 heads on 8, 100 keys behind 4,096 the first
// 45.3, 67.9 and 70.4, the second 61.0, 61.6 and 70.0.
bool paged_flash_gathers(const lvb_paged_desc* d, const PagedRoom& room) {
  if (d->prefix_len == 0) return false;
  const FlashSplit pre = paged_flash_split(d, room, kFlashPrefix, true);
  const FlashSplit own = paged_flash_split(d, room, kFlashOwn, true);
  // (not with parts beyond the workspace that the pool keeps: a part has all 256 rows of a pair)
  if (paged_flash_workspace(d, pre, kFlashPrefix, true) + paged_flash_workspace(d, own, kFlashOwn, true) >
      (size_t)512 << 20)
    return false;
  const double rows = (double)d->batch * (double)d->max_q * (double)d->heads_q;   // of the join
  const double parts_us = rows * (double)(pre.splits + own.splits) * (double)(d->head_dim + 2) * 8.0 / 5e6;
  return pre.us + own.us + parts_us + kJoinUs + kPassUs <
         paged_flash_split(d, room, kFlashOwn | kFlashPrefix, false).us;
}

// Items of different length are taken from a counter, when there are more than CTAs; a prefix's are
// alike and dealt in order. (The counter's reset is a step on the stream of its own: 10 rows over 144
// keys 15.1 us with it.)
bool paged_flash_counts(const lvb_paged_desc* d, FlashSplit fs, int parts, int sm_count) {
  return parts != kFlashPrefix && fs.cluster <= 1 &&
         paged_flash_items(d, parts) * fs.splits > std::max(1, sm_count);
}

int paged_flash_launch(const lvb_paged_desc* d, const PagedLayout& lay, const PagedSeqs& seqs,
                       const void* Q, const void* Kc, const void* Vc, void* O, float* lse, int parts,
                       bool joined, FlashSplit fs, void* ws, FlashWorkspace* out,
                       cudaStream_t stream, DeviceState* dev) {
  const char* op = "lvb_attention_paged";
  FlashParams p = {};
  p.seqs = seqs;
  p.Hq = (int)d->heads_q;
  p.Hkv = (int)d->heads_kv;
  p.group = p.Hq / p.Hkv;
  p.ppt = positions_per_tile(d);
  p.causal = d->causal ? 1 : 0;
  p.box = paged_box(d->page_size);
  p.own = (parts & kFlashOwn) ? 1 : 0;
  p.prefix = (parts & kFlashPrefix) ? (int)d->prefix_len : 0;
  p.all_rows = parts == kFlashPrefix ? 1 : 0;
  p.splits = fs.splits;
  p.pairs_per_seq = (int)tile_pairs(d, parts);
  p.cluster = fs.cluster > 1 ? fs.cluster : 0;
  p.late_wait = joined && !p.all_rows ? 1 : 0;
  p.store_parts = joined || fs.splits > fs.cluster ? 1 : 0;
  p.scale_log2 = d->scale * 1.4426950408889634f;
  p.O = O;
  p.o_st = lay.o[0];
  p.o_sh = lay.o[1];
  p.lse = lse;
  p.timeout_ns = wait_timeout_ns();
  const int64_t items = paged_flash_items(d, parts) * fs.splits;
  p.tile_o = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(ws) + kCounterBytes);
  const size_t stored = (size_t)(items / fs.cluster);
  p.tile_ml = p.tile_o + (p.store_parts ? stored * 256 * d->head_dim : 0);
  *out = FlashWorkspace{p.tile_o, p.tile_ml};
  CUtensorMap tq, tk, tv;
  {
    const uint64_t dims[3] = {(uint64_t)d->head_dim, (uint64_t)d->heads_q, (uint64_t)d->tokens};
    const uint64_t str[2] = {(uint64_t)lay.q[1], (uint64_t)lay.q[0]};
    const uint32_t box[3] = {64, (uint32_t)p.group, (uint32_t)p.ppt};
    int st = make_tmap_nd(&tq, Q, 2, 3, dims, str, box, op);
    if (st) return st;
  }
  int st = paged_kv_maps(&tk, &tv, d, lay, Kc, Vc, op);
  if (st) return st;
  const int ctas = p.cluster ? (int)items : (int)std::min<int64_t>(items, std::max(1, dev->sm_count));
  if (paged_flash_counts(d, fs, parts, dev->sm_count)) p.counter = reinterpret_cast<int*>(ws);
  if (d->head_dim == 128)
    return d->dtype == LVB_BF16 ? launch_flash<128, true>(tq, tk, tv, p, ctas, stream, dev)
                                : launch_flash<128, false>(tq, tk, tv, p, ctas, stream, dev);
  return d->dtype == LVB_BF16 ? launch_flash<64, true>(tq, tk, tv, p, ctas, stream, dev)
                              : launch_flash<64, false>(tq, tk, tv, p, ctas, stream, dev);
}

int merge_launch(const MergeParams& p, int D, bool bf16, cudaStream_t stream, DeviceState* dev) {
  const char* op = "lvb_attention_paged";
  const int rows = p.seqs.batch * p.seqs.max_q * p.Hq;
  const dim3 grid((unsigned)(((long long)rows * p.warps_per_row + 3) / 4));
  SmemAttr none;
  if (D == 128)
    return bf16 ? launch_serial(op, merge_kernel<128, true>, none, dev, grid, kMergeThreads, 0, stream, p, rows)
                : launch_serial(op, merge_kernel<128, false>, none, dev, grid, kMergeThreads, 0, stream, p, rows);
  return bf16 ? launch_serial(op, merge_kernel<64, true>, none, dev, grid, kMergeThreads, 0, stream, p, rows)
              : launch_serial(op, merge_kernel<64, false>, none, dev, grid, kMergeThreads, 0, stream, p, rows);
}

}  // namespace lvb
