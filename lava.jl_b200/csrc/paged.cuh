// paged.cuh — what the kernels on the paged KV cache share: the cache's description, a
// sequence's lengths read and checked on the device, and the TMA loads of a 128-key block
// that lies in several pages.
//
// Place p of sequence b is slot p % page_size of page table[b][p / page_size]; a shared prefix
// has a table of its own and stands before place 0 of every sequence. Lengths, tables and the
// queries' row offsets stay on the device (a captured graph is replayed while they change), so
// the kernels check them: a length outside the table counts as 0, a sequence whose query rows
// do not fit is left out, a page number outside the cache is read as zeros through the tensor
// map's bounds (and never written); each is recorded in the device status word.
#pragma once

#include <atomic>

#include "lvb_internal.h"

namespace lvb {

// A kernel's shared-memory attribute: per function and per device, set once (two threads setting
// it at once set the same value).
struct SmemAttr {
  static constexpr int kMaxDevices = 64;
  std::atomic<bool> set[kMaxDevices] = {};
};

// Launch with programmatic stream serialization: the kernel may be scheduled while the stream's
// previous kernel ends, and calls griddep_wait() before it touches global memory.
// cluster: CTAs per cluster (above 8 needs the function's leave too).
template <typename... P, typename... A>
int launch_cluster(const char* op, void (*kern)(P...), SmemAttr& attr, DeviceState* dev, dim3 grid,
                   int threads, size_t smem, int cluster, cudaStream_t stream, const A&... args) {
  if (smem > 48 * 1024 || cluster > 8) {
    const int dv = dev->device;
    const bool known = dv >= 0 && dv < SmemAttr::kMaxDevices;
    if (!known || !attr.set[dv].load(std::memory_order_acquire)) {
      const cudaError_t e =
          cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
      if (e != cudaSuccess) return fail_cuda(e, op, "cudaFuncSetAttribute");
      if (cluster > 0) {
        const cudaError_t e2 =
            cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e2 != cudaSuccess) return fail_cuda(e2, op, "cudaFuncSetAttribute");
      }
      if (known) attr.set[dv].store(true, std::memory_order_release);
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)cluster;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  return e == cudaSuccess ? LVB_OK : fail_cuda(e, op, "kernel launch");
}
template <typename... P, typename... A>
int launch_serial(const char* op, void (*kern)(P...), SmemAttr& attr, DeviceState* dev, dim3 grid,
                  int threads, size_t smem, cudaStream_t stream, const A&... args) {
  return launch_cluster(op, kern, attr, dev, grid, threads, smem, 0, stream, args...);
}

// Sites of bad device data in the status word (code LVB_ERR_INVALID_ARG).
constexpr int kBadLength = 81;   // seq_lens[b] negative or beyond the table's row
constexpr int kBadPage = 82;     // a page number outside 0..num_pages-1
constexpr int kBadRows = 83;     // cu_q not increasing, beyond `tokens`, or more than max_q rows

struct PagedSeqs {
  const int* table;            // [batch] rows of table_width page numbers
  const int* lens;             // [batch]
  const int* cu_q;             // [batch + 1], or NULL: max_q rows per sequence
  const int* prefix_table;
  long long table_stride;
  int table_width;
  int batch, max_q, tokens;
  int page_size, num_pages;
  int prefix_len;
  DevStatus* status;
};

__device__ __forceinline__ void report_bad(DevStatus* status, int where, int detail) {
  if (atomicCAS(&status->code, 0, 1 /* LVB_ERR_INVALID_ARG */) == 0) {
    status->where = where;
    status->block = blockIdx.x;
    status->detail = detail;
  }
}

// Element strides of a paged call with the packed ones filled in.
struct PagedLayout {
  long long q[2], o[2];     // token, head
  long long kc[3], vc[3];   // page, slot, head
};
PagedLayout paged_layout(const lvb_paged_desc& d);
int paged_kv_maps(CUtensorMap* tk, CUtensorMap* tv, const lvb_paged_desc* d, const PagedLayout& lay,
                  const void* Kc, const void* Vc, const char* op);
void paged_seqs(PagedSeqs* p, const lvb_paged_desc& d, const int32_t* table,
                const int32_t* seq_lens, const int32_t* cu_q, const int32_t* prefix_table,
                DeviceState* dev);
// How many CTAs with most of an SM's shared memory run at once: clusters of a size lie in one GPC, so
// their number depends on the chip's (measured here: 33 clusters of 4, 15 of 9, 7 of 16).
constexpr int kMostCluster = 16;
struct PagedRoom {
  int sms;
  int clusters[kMostCluster + 1];   // [size]
};

// Slots per TMA box: min(128, the largest power of two dividing the page size).
inline int paged_box(int64_t page_size) {
  int b = 8;
  while (b < 128 && page_size % (2 * b) == 0) b *= 2;
  return b;
}

int rope_launch(const lvb_rope_desc* d, const long long qs[3], const long long ks[3],
                const long long qos[3], const long long kos[3], const void* Q, const void* K,
                void* Qo, void* Ko, const int32_t* pos, const double* freqs, cudaStream_t stream,
                DeviceState* dev);
int append_launch(const lvb_append_desc* d, const PagedLayout& lay, const long long ks[2],
                  const long long vs[2], void* Kc, void* Vc, const void* K, const void* V,
                  const void* Q, void* Qo, const int32_t* table, const int32_t* seq_lens,
                  const int32_t* cu_q, const int32_t* pos, const double* freqs, cudaStream_t stream,
                  DeviceState* dev);

// Where the parts of a row's result lie, for the kernel that joins them (attn_paged_sm100.cu).
// A part is an unnormalised O row of D fp32, and the row's (reference maximum in log2 units, sum).
struct MergeParams {
  PagedSeqs seqs;
  int Hq, Hkv, group;
  // The key-range splits of the flash kernel's tiles: a part's rows are the 256 of a tile pair.
  const float* tile_o;         // [pair][Hkv][splits][256][D]
  const float* tile_ml;        // [pair][Hkv][splits][256][2]
  int tile_splits;             // 0: none
  int ppt;                     // positions per 128-row tile
  int pairs_per_seq;           // 0: pairs run over the tokens of the whole batch (the prefix)
  // The parts of a sequence's own keys beside a prefix's: the flash kernel's tiles again (laid out
  // as above, `own_pairs` per sequence), or the pieces of the decoding kernel: [slot][rows][D],
  // and where each item's pieces are.
  const float* own_o;
  const float* own_ml;
  int own_splits, own_pairs;   // own_splits 0: the decoding kernel's
  const int4* dec_tab;         // [batch·Hkv]; NULL: none
  int dec_rows;
  int dec_slots, dec_ctas;     // bounds of the table's entries
  int warps_per_row;           // 1, 2 or 4
  void* O;
  long long o_st, o_sh;
  float* lse;
};
int merge_launch(const MergeParams& p, int D, bool bf16, cudaStream_t stream, DeviceState* dev);

// The decoding kernel's table entry: (first slot, next CTA, last CTA, kind): the pieces are the
// first slot, then slot 2c of every CTA c from the next to the last.
enum { kItemDone = 0, kItemPieces = 1, kItemNoKeys = 2 };
struct DecodeWorkspace {
  float* part_o;
  float* part_ml;
  int4* tab;
  int rows, slots, ctas;
};
// Blocks that an item's start and end count for when the blocks are dealt out: the time of three
// 128-wide blocks, six 64-wide ones (measured on ragged batches: drafts over 64-wide heads 42.6 us
// with 1, 33.7 with 4, 32.3 with 6; 61 sequences of 128-wide heads 107.3 with 1, 103.7 with 3).
__host__ __device__ constexpr int paged_item_cost(int head_dim) { return 384 / head_dim; }
// CTAs per item when its blocks are split over a cluster, 0 when they are dealt to all CTAs.
int paged_decode_cluster(const lvb_paged_desc* d, const PagedRoom& room);
bool paged_decode_whole(const lvb_paged_desc* d, int sm_count);   // no item is cut (and `ws` NULL)
size_t paged_decode_workspace(const lvb_paged_desc* d, int sm_count, bool keep_parts);
// keep_parts: every item's result stays in the workspace for the join with a prefix's parts.
// after_prefix: the kernel before it is the same call's flash kernel over the prefix.
int paged_decode_launch(const lvb_paged_desc* d, const PagedLayout& lay, const PagedSeqs& seqs,
                        const void* Q, const void* Kc, const void* Vc, void* O, float* lse,
                        bool keep_parts, bool after_prefix, int cluster, void* ws,
                        DecodeWorkspace* out, cudaStream_t stream,
                        DeviceState* dev);

// The flash kernel over the prefix's keys, the sequences' own, or both one after the other.
struct FlashWorkspace {
  float* tile_o;
  float* tile_ml;
};
enum { kFlashOwn = 1, kFlashPrefix = 2 };
int64_t paged_flash_items(const lvb_paged_desc* d, int parts);
// Key ranges per tile pair, how many of them form a cluster (1: none), and the time this may take.
struct FlashSplit {
  int splits, cluster;
  double us;
};
// joined: the parts go to the join kernel in any case.
FlashSplit paged_flash_split(const lvb_paged_desc* d, const PagedRoom& room, int parts, bool joined);
bool paged_flash_gathers(const lvb_paged_desc* d, const PagedRoom& room);
size_t paged_flash_workspace(const lvb_paged_desc* d, FlashSplit fs, int parts, bool joined);
// Whether the first 4 bytes of `ws` are a counter, that the caller zeroes on the stream.
bool paged_flash_counts(const lvb_paged_desc* d, FlashSplit fs, int parts, int sm_count);
// The own pass of a joined call stands behind the prefix's: its CTAs take the SMs as the prefix's end
// (both fill an SM's shared memory), without a gap between the two kernels.
int paged_flash_launch(const lvb_paged_desc* d, const PagedLayout& lay, const PagedSeqs& seqs,
                       const void* Q, const void* Kc, const void* Vc, void* O, float* lse, int parts,
                       bool joined, FlashSplit fs, void* ws, FlashWorkspace* out,
                       cudaStream_t stream, DeviceState* dev);

// Log2 units that a weight of P is held above its value relative to the row's reference maximum. fp16:
// 2^6, away from the subnormals, so that a weight is lost (in the product with V, not in the sum) below
// 2^-31 of the reference and not below 2^-25, where a long flat tail still counts; a score may exceed
// the reference by 2^8, and 2^14 is below the largest fp16. A part's m is lowered by as much.
template <bool BF16>
constexpr float kWeightShift = BF16 ? 0.f : 6.f;

struct SeqInfo {
  int tok0;   // first query row
  int qlen;   // query rows (0: the sequence takes no part)
  int len;    // keys in the cache
};

// Sequence b from its length and row offsets as the lists have them.
__device__ __forceinline__ SeqInfo seq_checked(const PagedSeqs& p, int b, int len, int row0, int row1) {
  SeqInfo s{row0, 0, len};
  const long long q = (long long)row1 - row0;
  if (q < 0 || q > p.max_q || row0 < 0 || row1 > p.tokens) report_bad(p.status, kBadRows, b);
  else s.qlen = (int)q;
  if (len < 0 || len > (long long)p.table_width * p.page_size) {
    report_bad(p.status, kBadLength, b);
    s.len = 0;
  }
  return s;
}
__device__ __forceinline__ SeqInfo seq_info(const PagedSeqs& p, int b) {
  const int row0 = p.cu_q ? p.cu_q[b] : b * p.max_q;
  const int row1 = p.cu_q ? p.cu_q[b + 1] : row0 + p.max_q;
  return seq_checked(p, b, p.lens[b], row0, row1);
}

// ----------------------------------------------------------------------------------------
// One 128-key block by TMA. The box is `box` = min(128, the largest power of two dividing the
// page size) slots high and 64 elements (128 bytes) wide, so 128/box boxes times D/64 chunks
// make a block: at most 32, one per lane of the producing warp. Lane i's box holds keys
// sub·box .. of chunk c. Boxes without a valid key are not loaded.
// ----------------------------------------------------------------------------------------
template <int D>
struct BlockLane {
  static constexpr int kCh = D / 64;
  int sub, c;
  bool in;
  __device__ __forceinline__ BlockLane(int lane, int box) {
    sub = lane / kCh;
    c = lane - sub * kCh;
    in = sub * box < 128;
  }
};

// The page and slot of a lane's box.
struct BoxAt {
  int page, slot;
  bool on;            // the box holds a valid key
};

// The boxes of one block after the other of a run of `n` keys whose pages are r[0 ..], worked out by
// a whole warp. The table entries come 32 at a time, one
// per lane, with the next 32 on their way, and a box's entry is fetched from its lane: under a
// saturated memory system a table load takes as long as several blocks (measured: every fourth
// block of a 64-slot-page cache waited 3,000-5,000 clk for its entries when they were loaded one
// block ahead). Place p + 128 is `whole` pages and `rest` slots on, without a division.
template <int D>
struct BoxWalk {
  const int* row;
  int key, len, i, slot;
  int page_size, whole, rest;
  int w0, last;       // first entry of the window; the run's last entry
  int cur, nxt;       // this lane's entries of the window and of the one behind it
  bool in;
  __device__ __forceinline__ int entry(int k) const { return k <= last ? row[k] : 0; }
  // `entries`: the run's first 32 entries from block kb on, when they are in shared memory already.
  __device__ __forceinline__ void start(const BlockLane<D>& bl, const int* r, int kb, int n, int box,
                                        int psize, const int* entries = nullptr) {
    row = r;
    len = n;
    in = bl.in;
    page_size = psize;
    key = kb * 128 + bl.sub * box;
    i = key / psize;
    slot = key - i * psize;
    whole = 128 / psize;
    rest = 128 - whole * psize;
    w0 = __shfl_sync(0xffffffffu, i, 0);
    last = (n - 1) / psize;
    cur = entries ? entries[lane_id()] : entry(w0 + (int)lane_id());
    nxt = entry(w0 + 32 + (int)lane_id());
  }
  __device__ __forceinline__ BoxAt take() {
    // the lanes' entries lie within two windows of lane 0's; the second is only looked at (and so
    // waited for) once a lane needs it
    const int at0 = i - w0;
    int page = __shfl_sync(0xffffffffu, cur, at0 & 31);
    if (__any_sync(0xffffffffu, at0 >= 32)) {
      const int c = __shfl_sync(0xffffffffu, nxt, at0 & 31);
      if (at0 >= 32) page = c;
    }
    const BoxAt at{page, slot, in && key < len};
    key += 128;
    i += whole;
    slot += rest;
    if (slot >= page_size) {
      slot -= page_size;
      ++i;
    }
    if (__shfl_sync(0xffffffffu, i, 0) - w0 >= 32) {
      w0 += 32;
      cur = nxt;
      nxt = entry(w0 + 32 + (int)lane_id());
    }
    return at;
  }
};

// Issue one block's loads into `dst` ([D/64 chunks][128 rows][128 B], 128-byte swizzle) on
// `bar`; the whole warp calls it. A bad page number becomes num_pages, which the tensor map
// reads as zeros.
template <int D>
__device__ __forceinline__ void load_block(uint8_t* dst, const CUtensorMap* tm,
                                           const BlockLane<D>& bl, BoxAt at, int box, int hk,
                                           uint64_t* bar, const PagedSeqs& p) {
  const unsigned on = __ballot_sync(0xffffffffu, at.on);
  if (lane_id() == 0) bar_arrive_expect_tx(bar, (uint32_t)__popc(on) * box * 128u);
  __syncwarp();
  if (at.on) {
    if (at.page < 0 || at.page >= p.num_pages) {
      report_bad(p.status, kBadPage, at.page);
      at.page = p.num_pages;
    }
    tma_load_4d(dst + bl.c * (128 * 128) + bl.sub * box * 128, tm, bl.c * 64, at.slot, hk, at.page,
                bar);
  }
  __syncwarp();
}

// A 4-byte copy to shared memory that the thread does not wait for, and the arrival (one of the
// barrier's count) once this thread's copies so far have landed.
__device__ __forceinline__ void copy_async4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Loads from a CTA of the cluster (a shared::cluster address, see mapa_shared).
__device__ __forceinline__ float ld_cluster_f32(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster_f32x2(uint32_t a) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(a)
               : "memory");
  return v;
}

// A wait by a whole warp that tests once before it suspends: the phase is often complete already,
// and the suspending form costs a few hundred cycles even then.
__device__ __forceinline__ bool wait_soon_warp(uint64_t* bar, uint32_t parity, const WaitGuard& g,
                                               int where, int detail) {
  const bool ok = bar_test_wait(smem_u32(bar), parity);
  if (__all_sync(0xffffffffu, ok)) return true;
  return wait_bar_warp(bar, parity, g, where, detail);
}

// Zero rows [valid, 128) of a block ([D/64 chunks][128 rows][128 B]; whole rows, so the swizzle
// plays no part) by one warp, and make the stores visible to the tensor core. What a page holds
// behind a sequence's last place is stale (possibly infinite or NaN), and 0·NaN would reach the
// sum through P·V although P is 0 there.
template <int D>
__device__ __forceinline__ void zero_tail(uint32_t block_saddr, int valid) {
  const int lane = lane_id();
  for (int c = 0; c < D / 64; ++c)
    for (int i = valid * 8 + lane; i < 128 * 8; i += 32)
      st_shared_v4(block_saddr + c * (128 * 128) + i * 16, 0, 0, 0, 0);
  fence_proxy_async_smem();
  __syncwarp();
}

}  // namespace lvb
