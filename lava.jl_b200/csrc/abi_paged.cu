// abi_paged.cu — the extern "C" surface of position rotation, the paged KV cache's append and the
// attention over it: argument validation, planning and launch order.
#include <cmath>
#include <cstring>

#include <algorithm>
#include <mutex>

#include "paged.cuh"

namespace lvb {

PagedLayout paged_layout(const lvb_paged_desc& d) {
  PagedLayout l;
  auto two = [&](const int64_t* s, long long* o) {
    const bool packed = s[0] == 0 && s[1] == 0;
    o[0] = packed ? d.heads_q * d.head_dim : s[0];
    o[1] = packed ? d.head_dim : s[1];
  };
  auto three = [&](const int64_t* s, long long* o) {
    const bool packed = s[0] == 0 && s[1] == 0 && s[2] == 0;
    o[0] = packed ? d.page_size * d.heads_kv * d.head_dim : s[0];
    o[1] = packed ? d.heads_kv * d.head_dim : s[1];
    o[2] = packed ? d.head_dim : s[2];
  };
  two(d.q_stride, l.q);
  two(d.o_stride, l.o);
  three(d.kc_stride, l.kc);
  three(d.vc_stride, l.vc);
  return l;
}

void paged_seqs(PagedSeqs* p, const lvb_paged_desc& d, const int32_t* table,
                const int32_t* seq_lens, const int32_t* cu_q, const int32_t* prefix_table,
                DeviceState* dev) {
  p->table = table;
  p->lens = seq_lens;
  p->cu_q = cu_q;
  p->prefix_table = prefix_table;
  p->table_stride = d.table_stride ? d.table_stride : d.table_width;
  p->table_width = (int)d.table_width;
  p->batch = (int)d.batch;
  p->max_q = (int)d.max_q;
  p->tokens = (int)d.tokens;
  p->page_size = (int)d.page_size;
  p->num_pages = (int)d.num_pages;
  p->prefix_len = (int)d.prefix_len;
  p->status = dev->status;
}

// 4-D maps over the cache: (64 of head_dim, slots of a page, KV head, page).
int paged_kv_maps(CUtensorMap* tk, CUtensorMap* tv, const lvb_paged_desc* d, const PagedLayout& lay,
                  const void* Kc, const void* Vc, const char* op) {
  const uint64_t dims[4] = {(uint64_t)d->head_dim, (uint64_t)d->page_size, (uint64_t)d->heads_kv,
                            (uint64_t)d->num_pages};
  const uint32_t box[4] = {64, (uint32_t)paged_box(d->page_size), 1, 1};
  const uint64_t sk[3] = {(uint64_t)lay.kc[1], (uint64_t)lay.kc[2], (uint64_t)lay.kc[0]};
  const uint64_t sv[3] = {(uint64_t)lay.vc[1], (uint64_t)lay.vc[2], (uint64_t)lay.vc[0]};
  // A head's row may lie between other heads': fetch no more than it.
  const int fetch = (int)d->head_dim * 2;
  int st = make_tmap_nd(tk, Kc, 2, 4, dims, sk, box, op, fetch);
  if (st) return st;
  return make_tmap_nd(tv, Vc, 2, 4, dims, sv, box, op, fetch);
}

namespace {

constexpr int64_t kMostKeys = 1LL << 30;   // of a sequence or a prefix

// `n` element strides of a 16-bit or 32-bit tensor whose head_dim is contiguous: all zero
// (packed), or each a multiple of 16 bytes and at least head_dim where its extent is above 1.
int check_strides(const char* op, const char* what, const int64_t* s, const int64_t* extent, int n,
                  int64_t head_dim, int esize) {
  bool packed = true;
  for (int i = 0; i < n; ++i) packed = packed && s[i] == 0;
  if (packed) return LVB_OK;
  for (int i = 0; i < n; ++i) {
    if (s[i] < 0 || (extent[i] > 1 && s[i] < head_dim))
      return fail(LVB_ERR_INVALID_ARG, op, std::string(what) + ": stride below head_dim");
    if ((s[i] * esize) % 16)
      return fail(LVB_ERR_UNSUPPORTED, op, std::string(what) + ": strides must be multiples of 16 bytes");
  }
  return LVB_OK;
}

int check_rotation(const char* op, const lvb_rotation& r, int64_t head_dim) {
  if (r.pairs < 0 || r.pairs % 8 || 2 * (int64_t)r.pairs > head_dim)
    return fail(LVB_ERR_UNSUPPORTED, op, "pairs must be a multiple of 8 and at most head_dim / 2");
  if (r.layout != LVB_ROPE_HALVES && r.layout != LVB_ROPE_PAIRS)
    return fail(LVB_ERR_INVALID_ARG, op, "unknown rotation layout");
  if (r.n_axes < 1 || r.n_axes > LVB_ROPE_MAX_AXES)
    return fail(LVB_ERR_INVALID_ARG, op, "n_axes must be 1..4");
  int64_t sum = 0;
  for (int a = 0; a < r.n_axes; ++a) {
    if (r.sections[a] < 0) return fail(LVB_ERR_INVALID_ARG, op, "negative section");
    sum += r.sections[a];
  }
  if (sum != r.pairs)
    return fail(LVB_ERR_INVALID_ARG, op, "the sections' pairs must add up to `pairs`");
  return LVB_OK;
}

// What the append and the attention ask of the cache and the batch.
int check_paged(const char* op, const lvb_paged_desc* d) {
  if (!d) return fail(LVB_ERR_INVALID_ARG, op, "descriptor is NULL");
  if (d->batch < 0 || d->heads_q < 0 || d->heads_kv < 0 || d->tokens < 0 || d->max_q < 0 ||
      d->table_width < 0 || d->prefix_len < 0)
    return fail(LVB_ERR_INVALID_ARG, op, "negative extent");
  if (d->dtype != LVB_F16 && d->dtype != LVB_BF16)
    return fail(LVB_ERR_UNSUPPORTED, op, std::string("no kernel for ") + dtype_name(d->dtype),
                "Float16 or BFloat16");
  if (d->heads_kv == 0 || d->heads_q % d->heads_kv)
    return fail(LVB_ERR_INVALID_ARG, op, "heads_q must be a multiple of heads_kv");
  if (d->head_dim != 64 && d->head_dim != 128)
    return fail(LVB_ERR_UNSUPPORTED, op, "head_dim must be 64 or 128");
  if (d->page_size <= 0 || d->page_size % 8)
    return fail(LVB_ERR_UNSUPPORTED, op, "page_size must be a positive multiple of 8");
  if (d->num_pages < 1) return fail(LVB_ERR_INVALID_ARG, op, "the cache has no page");
  if (d->table_stride < 0 || (d->table_stride > 0 && d->table_stride < d->table_width))
    return fail(LVB_ERR_INVALID_ARG, op, "table_stride < table_width");
  if (d->page_size > kMostKeys || d->table_width > kMostKeys / d->page_size ||
      d->prefix_len > kMostKeys)
    return fail(LVB_ERR_UNSUPPORTED, op, "more than 2^30 keys per sequence");
  if (d->num_pages >= INT32_MAX || d->tokens > INT32_MAX || d->max_q > INT32_MAX ||
      d->batch > INT32_MAX || d->heads_q > 65535 || d->heads_kv > INT32_MAX / 2 ||
      d->batch * d->heads_kv > INT32_MAX ||
      (d->batch > 0 && d->max_q > INT32_MAX / d->batch))
    return fail(LVB_ERR_UNSUPPORTED, op, "extent above 2^31-1", "split the batch");
  const int64_t cache[3] = {d->num_pages, d->page_size, d->heads_kv};
  const int64_t rows[2] = {d->tokens, d->heads_q};
  int st;
  if ((st = check_strides(op, "K cache", d->kc_stride, cache, 3, d->head_dim, 2))) return st;
  if ((st = check_strides(op, "V cache", d->vc_stride, cache, 3, d->head_dim, 2))) return st;
  if ((st = check_strides(op, "Q", d->q_stride, rows, 2, d->head_dim, 2))) return st;
  return check_strides(op, "the result", d->o_stride, rows, 2, d->head_dim, 2);
}

int check_lists(const char* op, const lvb_paged_desc* d, const int32_t* table,
                const int32_t* seq_lens, const int32_t* cu_q, const int32_t* prefix_table) {
  if (!seq_lens || (d->table_width > 0 && !table))
    return fail(LVB_ERR_INVALID_ARG, op, "block table or seq_lens is NULL");
  if (!cu_q && d->tokens != d->batch * d->max_q)
    return fail(LVB_ERR_INVALID_ARG, op, "without cu_q, tokens must be batch·max_q");
  if (((uintptr_t)table | (uintptr_t)seq_lens | (uintptr_t)cu_q | (uintptr_t)prefix_table) % 4)
    return fail(LVB_ERR_INVALID_ARG, op, "pointer not aligned to its element size");
  return LVB_OK;
}

// The decoding kernel's products hold 16 rows. (More rows in wider products, with twice the softmax
// per key, took 125 us at 24 rows over 8·8 times 16,384 keys, the flash kernel 106; 28 and 21 over
// 1,000 keys, 15.8 and 10.6 over 300; at 16 rows 97 and 103, 16.3 and 20.1, 9.6 and 10.7. All of that
// at 64 items, which the flash kernel splits in two key ranges; from 75 items on it does not, see
// paged_flash_split, and the wider products were not measured there.)
bool use_decode(const lvb_paged_desc* d) {
  return (d->heads_q / d->heads_kv) * d->max_q <= 16;
}

// The decoding kernel deals units, an item's being its own key blocks and its cost, and counts them in
// 32 bits: their total, and the total with one CTA's share behind it (at most half of it and a unit
// when there are two CTAs; with one there is no second share). The prefix's blocks are not among
// them but where paged_decode_whole bounds their number by the SMs'.
bool units_fit(const lvb_paged_desc* d) {
  const int64_t units = (d->table_width * d->page_size + 127) / 128 + paged_item_cost((int)d->head_dim);
  return d->batch * d->heads_kv <= INT32_MAX / 3 * 2 / units;
}

size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// The numbers of clusters as measured on a B200, for a plan without a device, scaled to `sm_count`.
PagedRoom static_room(int sm_count) {
  static const int k148[kMostCluster + 1] = {0, 148, 74, 45, 33, 26, 22, 15, 15, 15, 11, 7, 7, 7, 7, 7, 7};
  PagedRoom r;
  r.sms = sm_count;
  for (int c = 0; c <= kMostCluster; ++c) r.clusters[c] = (int)((int64_t)k148[c] * sm_count / 148);
  return r;
}

__global__ void cluster_probe_kernel() {}

// The device's own numbers, asked once.
int device_room(DeviceState* dev, PagedRoom* out, const char* op) {
  struct Asked {
    std::once_flag once;
    PagedRoom room;
  };
  static Asked asked[64];
  if (dev->device < 0 || dev->device >= 64) {
    *out = static_room(dev->sm_count);
    return LVB_OK;
  }
  Asked& a = asked[dev->device];
  std::call_once(a.once, [&] {
    a.room = static_room(dev->sm_count);
    const int smem = 220 * 1024;
    if (cudaFuncSetAttribute(cluster_probe_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
        cudaFuncSetAttribute(cluster_probe_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) {
      cudaGetLastError();
      return;
    }
    for (int c = 2; c <= kMostCluster; ++c) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(c);
      cfg.blockDim = dim3(384);
      cfg.dynamicSmemBytes = smem;
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim.x = (unsigned)c;
      at[0].val.clusterDim.y = 1;
      at[0].val.clusterDim.z = 1;
      cfg.attrs = at;
      cfg.numAttrs = 1;
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, cluster_probe_kernel, &cfg) == cudaSuccess) {
        a.room.clusters[c] = n;
      } else {
        cudaGetLastError();
        a.room.clusters[c] = 0;      // such clusters are not used
      }
    }
  });
  *out = a.room;
  return LVB_OK;
}

// Workspace of a planned call: the flash kernel's over the prefix, then what the sequences' own
// keys need.
size_t prefix_bytes(const lvb_paged_desc* d, const lvb_paged_plan& pl) {
  if (!pl.prefix_splits) return 0;
  return up256(paged_flash_workspace(d, FlashSplit{pl.prefix_splits, 1, 0.0}, kFlashPrefix, true));
}

int plan_paged(const lvb_paged_desc* d, const PagedRoom& room, lvb_paged_plan* out) {
  const char* op = "lvb_attention_paged";
  std::memset(out, 0, sizeof *out);
  out->splits = 1;
  if (d->batch == 0 || d->tokens == 0 || d->max_q == 0 || d->heads_q == 0) return LVB_OK;
  const bool decode = use_decode(d);
  out->kernel = decode ? LVB_PAGED_DECODE : LVB_PAGED_FLASH;
  if (paged_flash_items(d, kFlashOwn) > INT32_MAX - 65536)
    return fail(LVB_ERR_UNSUPPORTED, op, "more than 2^31 query tiles", "split the batch");
  if (decode && ((out->cluster = paged_decode_cluster(d, room)) > 0 || paged_decode_whole(d, room.sms))) {
    out->launches = 1;      // no parts in memory
    return LVB_OK;
  }
  if (d->prefix_len && (decode || paged_flash_gathers(d, room)))
    out->prefix_splits = paged_flash_split(d, room, kFlashPrefix, true).splits;
  const bool joined = out->prefix_splits > 0;
  if (decode) {
    // (rows of the join, counted in 32 bits)
    if ((double)d->batch * (double)d->max_q * (double)d->heads_q > (double)(INT32_MAX / 4))
      return fail(LVB_ERR_UNSUPPORTED, op, "more than 2^29 query rows", "split the batch");
    out->launches = joined ? 3 : 2;
    out->workspace_bytes =
        (int64_t)(prefix_bytes(d, *out) + paged_decode_workspace(d, room.sms, joined));
    return LVB_OK;
  }
  const int parts = kFlashOwn | (d->prefix_len && !joined ? kFlashPrefix : 0);
  const FlashSplit fs = paged_flash_split(d, room, parts, joined);
  out->splits = fs.splits;
  out->cluster = fs.cluster > 1 ? fs.cluster : 0;
  out->launches = joined ? 3 : fs.splits > fs.cluster ? 2 : 1;
  out->workspace_bytes =
      (int64_t)(prefix_bytes(d, *out) + paged_flash_workspace(d, fs, parts, joined));
  return LVB_OK;
}

}  // namespace
}  // namespace lvb

using namespace lvb;

extern "C" {

// ---------------------------------------------------------------------------------------
// Rotation
// ---------------------------------------------------------------------------------------
int lvb_rope_check(const lvb_rope_desc* d) {
  const char* op = "lvb_rope";
  if (!d) return fail(LVB_ERR_INVALID_ARG, op, "descriptor is NULL");
  if (d->batch < 0 || d->heads_q < 0 || d->heads_kv < 0 || d->seq < 0)
    return fail(LVB_ERR_INVALID_ARG, op, "negative extent");
  if (d->dtype != LVB_F16 && d->dtype != LVB_BF16 && d->dtype != LVB_F32)
    return fail(LVB_ERR_UNSUPPORTED, op, std::string("no kernel for ") + dtype_name(d->dtype),
                "Float16, BFloat16 or Float32");
  if (d->head_dim <= 0 || d->head_dim % 16 || d->head_dim > 512)
    return fail(LVB_ERR_UNSUPPORTED, op, "head_dim must be a multiple of 16, at most 512");
  if (d->seq > INT32_MAX || d->batch > 65535 || d->heads_q > 65535 || d->heads_kv > 65535)
    return fail(LVB_ERR_UNSUPPORTED, op, "more than 2^31-1 positions, 65535 sequences or heads",
                "split the batch");
  int st = check_rotation(op, d->rot, d->head_dim);
  if (st) return st;
  if (d->rot.pairs == 0) return fail(LVB_ERR_INVALID_ARG, op, "pairs must be at least 8");
  const int es = dtype_size(d->dtype);
  const int64_t eq[3] = {d->batch, d->heads_q, d->seq}, ek[3] = {d->batch, d->heads_kv, d->seq};
  if ((st = check_strides(op, "Q", d->q_stride, eq, 3, d->head_dim, es))) return st;
  if ((st = check_strides(op, "K", d->k_stride, ek, 3, d->head_dim, es))) return st;
  if ((st = check_strides(op, "rotated Q", d->qo_stride, eq, 3, d->head_dim, es))) return st;
  return check_strides(op, "rotated K", d->ko_stride, ek, 3, d->head_dim, es);
}

int lvb_rope(const lvb_rope_desc* d, const void* Q, const void* K, void* Qo, void* Ko,
             const int32_t* pos, const double* freqs, void* stream) {
  const char* op = "lvb_rope";
  int st = lvb_rope_check(d);
  if (st) return st;
  if (d->batch == 0 || d->seq == 0 || d->heads_q + d->heads_kv == 0) return LVB_OK;
  if ((d->heads_q && (!Q || !Qo)) || (d->heads_kv && (!K || !Ko)) || !pos || !freqs)
    return fail(LVB_ERR_INVALID_ARG, op, "a tensor, pos or freqs is NULL");
  if (((uintptr_t)Q | (uintptr_t)K | (uintptr_t)Qo | (uintptr_t)Ko) % 16)
    return fail(LVB_ERR_UNSUPPORTED, op, "tensors must start on 16-byte boundaries");
  if ((uintptr_t)pos % 4 || (uintptr_t)freqs % 8)
    return fail(LVB_ERR_INVALID_ARG, op, "pointer not aligned to its element size");
  DeviceState* dev = current_device_state(op);
  if (!dev) return LVB_ERR_NO_DEVICE;
  long long s[4][3];
  const int64_t* given[4] = {d->q_stride, d->k_stride, d->qo_stride, d->ko_stride};
  for (int t = 0; t < 4; ++t) {
    const int64_t* g = given[t];
    const int64_t H = t % 2 ? d->heads_kv : d->heads_q;
    const bool packed = g[0] == 0 && g[1] == 0 && g[2] == 0;
    s[t][0] = packed ? H * d->seq * d->head_dim : g[0];
    s[t][1] = packed ? d->seq * d->head_dim : g[1];
    s[t][2] = packed ? d->head_dim : g[2];
  }
  return rope_launch(d, s[0], s[1], s[2], s[3], Q, K, Qo, Ko, pos, freqs,
                     reinterpret_cast<cudaStream_t>(stream), dev);
}

// ---------------------------------------------------------------------------------------
// Append
// ---------------------------------------------------------------------------------------
int lvb_kv_append_check(const lvb_append_desc* d) {
  const char* op = "lvb_kv_append";
  if (!d) return fail(LVB_ERR_INVALID_ARG, op, "descriptor is NULL");
  int st = check_paged(op, &d->paged);
  if (st) return st;
  const int64_t rows[2] = {d->paged.tokens, d->paged.heads_kv};
  if ((st = check_strides(op, "K", d->k_stride, rows, 2, d->paged.head_dim, 2))) return st;
  if ((st = check_strides(op, "V", d->v_stride, rows, 2, d->paged.head_dim, 2))) return st;
  return d->rot.pairs == 0 ? LVB_OK : check_rotation(op, d->rot, d->paged.head_dim);
}

int lvb_kv_append(const lvb_append_desc* d, void* Kc, void* Vc, const void* K, const void* V,
                  const void* Q, void* Qo, const int32_t* table, const int32_t* seq_lens,
                  const int32_t* cu_q, const int32_t* pos, const double* freqs, void* stream) {
  const char* op = "lvb_kv_append";
  int st = lvb_kv_append_check(d);
  if (st) return st;
  const lvb_paged_desc& g = d->paged;
  if (g.batch == 0 || g.tokens == 0 || g.max_q == 0) return LVB_OK;
  if (!Kc || !Vc || !K || !V || (!Q != !Qo))
    return fail(LVB_ERR_INVALID_ARG, op, "K, V, a cache or one of Q and Qo is NULL");
  if ((st = check_lists(op, &g, table, seq_lens, cu_q, nullptr))) return st;
  if (d->rot.pairs == 0 && Q)
    return fail(LVB_ERR_INVALID_ARG, op, "Q without a rotation", "pairs is 0");
  if (d->rot.pairs > 0 && !freqs) return fail(LVB_ERR_INVALID_ARG, op, "freqs is NULL");
  if (d->rot.pairs > 0 && !pos && d->rot.n_axes != 1)
    return fail(LVB_ERR_INVALID_ARG, op, "pos is NULL with several axes",
                "only one axis can count the places");
  if (((uintptr_t)Kc | (uintptr_t)Vc | (uintptr_t)K | (uintptr_t)V | (uintptr_t)Q | (uintptr_t)Qo) % 16)
    return fail(LVB_ERR_UNSUPPORTED, op, "tensors must start on 16-byte boundaries");
  if ((uintptr_t)pos % 4 || (uintptr_t)freqs % 8)
    return fail(LVB_ERR_INVALID_ARG, op, "pointer not aligned to its element size");
  DeviceState* dev = current_device_state(op);
  if (!dev) return LVB_ERR_NO_DEVICE;
  long long ks[2], vs[2];
  for (int t = 0; t < 2; ++t) {
    const int64_t* s = t ? d->v_stride : d->k_stride;
    long long* o = t ? vs : ks;
    const bool packed = s[0] == 0 && s[1] == 0;
    o[0] = packed ? g.heads_kv * g.head_dim : s[0];
    o[1] = packed ? g.head_dim : s[1];
  }
  return append_launch(d, paged_layout(g), ks, vs, Kc, Vc, K, V, Q, Qo, table, seq_lens, cu_q, pos,
                       freqs, reinterpret_cast<cudaStream_t>(stream), dev);
}

// ---------------------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------------------
int lvb_attention_paged_check(const lvb_paged_desc* d) {
  const char* op = "lvb_attention_paged";
  int st = check_paged(op, d);
  if (st) return st;
  if (!(d->scale > 0.0f) || std::isinf(d->scale))
    return fail(LVB_ERR_INVALID_ARG, op, "scale must be a positive finite number");
  if (d->heads_q / d->heads_kv > 128)
    return fail(LVB_ERR_UNSUPPORTED, op, "more than 128 query heads per KV head");
  if (use_decode(d) && !units_fit(d))
    return fail(LVB_ERR_UNSUPPORTED, op, "more than 2^30 key blocks and items in the tables",
                "split the batch");
  return LVB_OK;
}

int lvb_attention_paged_plan_for(const lvb_paged_desc* d, int32_t sm_count, lvb_paged_plan* out) {
  const char* op = "lvb_attention_paged";
  int st = lvb_attention_paged_check(d);
  if (st) return st;
  if (!out) return fail(LVB_ERR_INVALID_ARG, op, "plan is NULL");
  return plan_paged(d, static_room(sm_count > 0 ? sm_count : 148), out);
}

int lvb_attention_paged(const lvb_paged_desc* d, const void* Q, const void* Kc, const void* Vc,
                        const int32_t* table, const int32_t* seq_lens, const int32_t* cu_q,
                        const int32_t* prefix_table, void* O, float* lse, void* stream) {
  const char* op = "lvb_attention_paged";
  int st = lvb_attention_paged_check(d);
  if (st) return st;
  if (d->batch == 0 || d->tokens == 0 || d->max_q == 0 || d->heads_q == 0) return LVB_OK;
  if (!Q || !O || !Kc || !Vc) return fail(LVB_ERR_INVALID_ARG, op, "Q, O or a cache is NULL");
  if ((st = check_lists(op, d, table, seq_lens, cu_q, prefix_table))) return st;
  if (d->prefix_len && !prefix_table)
    return fail(LVB_ERR_INVALID_ARG, op, "prefix_table is NULL", "prefix_len is above 0");
  if (((uintptr_t)Q | (uintptr_t)O | (uintptr_t)Kc | (uintptr_t)Vc) % 16)
    return fail(LVB_ERR_UNSUPPORTED, op, "tensors must start on 16-byte boundaries");
  if ((uintptr_t)lse % 4) return fail(LVB_ERR_INVALID_ARG, op, "lse not aligned to its element size");
  DeviceState* dev = current_device_state(op);
  if (!dev) return LVB_ERR_NO_DEVICE;
  lvb_paged_plan pl;
  PagedRoom room;
  if ((st = device_room(dev, &room, op)) || (st = plan_paged(d, room, &pl))) return st;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const PagedLayout lay = paged_layout(*d);
  MergeParams mp = {};
  paged_seqs(&mp.seqs, *d, table, seq_lens, cu_q, prefix_table, dev);
  mp.Hq = (int)d->heads_q;
  mp.Hkv = (int)d->heads_kv;
  mp.group = mp.Hq / mp.Hkv;
  mp.ppt = 128 / mp.group;
  mp.O = O;
  mp.o_st = lay.o[0];
  mp.o_sh = lay.o[1];
  mp.lse = lse;
  uint8_t* ws = nullptr;
  if (pl.kernel == LVB_PAGED_DECODE && pl.launches == 1) {
    DecodeWorkspace none = {};
    return paged_decode_launch(d, lay, mp.seqs, Q, Kc, Vc, O, lse, false, false, pl.cluster, ws, &none,
                               s, dev);
  }
  cudaError_t e = workspace_alloc(dev, reinterpret_cast<void**>(&ws), (size_t)pl.workspace_bytes, s);
  if (e != cudaSuccess) return fail_cuda(e, op, "workspace allocation");
  const bool bf16 = d->dtype == LVB_BF16;
  const bool joined = pl.prefix_splits > 0;
  uint8_t* own_ws = ws + prefix_bytes(d, pl);
  const int parts = kFlashOwn | (d->prefix_len && !joined ? kFlashPrefix : 0);
  const FlashSplit fs{pl.splits, std::max(1, pl.cluster), 0.0};
  // (before the prefix's kernel, so that nothing stands between it and the one behind it)
  if (pl.kernel == LVB_PAGED_FLASH && paged_flash_counts(d, fs, parts, dev->sm_count)) {
    e = cudaMemsetAsync(own_ws, 0, sizeof(int), s);
    if (e != cudaSuccess) st = fail_cuda(e, op, "work counter reset");
  }
  FlashWorkspace fw = {};
  if (joined && st == LVB_OK) {
    st = paged_flash_launch(d, lay, mp.seqs, Q, Kc, Vc, O, lse, kFlashPrefix, true,
                            FlashSplit{pl.prefix_splits, 1, 0.0}, ws, &fw, s, dev);
    mp.tile_o = fw.tile_o;
    mp.tile_ml = fw.tile_ml;
    mp.tile_splits = pl.prefix_splits;
  }
  int pieces = mp.tile_splits;      // parts of a row, about
  if (pl.kernel == LVB_PAGED_DECODE) {
    DecodeWorkspace dw = {};
    if (st == LVB_OK)
      st = paged_decode_launch(d, lay, mp.seqs, Q, Kc, Vc, O, lse, joined, joined, 0, own_ws, &dw, s,
                               dev);
    mp.own_o = dw.part_o;
    mp.own_ml = dw.part_ml;
    mp.dec_tab = dw.tab;
    mp.dec_rows = dw.rows;
    mp.dec_slots = dw.slots;
    mp.dec_ctas = dw.ctas;
    // about as many pieces per item as there are CTAs for each, and one more
    pieces += dw.ctas / (int)(d->batch * d->heads_kv) + 2;
  } else {
    if (st == LVB_OK)
      st = paged_flash_launch(d, lay, mp.seqs, Q, Kc, Vc, O, lse, parts, joined, fs, own_ws, &fw, s, dev);
    const int groups = fs.splits / fs.cluster;
    const int pairs = (int)((d->max_q + 2 * mp.ppt - 1) / (2 * mp.ppt));
    if (joined) {
      mp.own_o = fw.tile_o;
      mp.own_ml = fw.tile_ml;
      mp.own_splits = groups;
      mp.own_pairs = pairs;
    } else {
      mp.tile_o = fw.tile_o;
      mp.tile_ml = fw.tile_ml;
      mp.tile_splits = groups;
      mp.pairs_per_seq = pairs;
    }
    pieces += groups;
  }
  if (pl.kernel == LVB_PAGED_DECODE || joined || mp.tile_splits > 1) {
    mp.warps_per_row = pieces <= 8 ? 1 : pieces <= 16 ? 2 : 4;
    if (st == LVB_OK) st = merge_launch(mp, (int)d->head_dim, bf16, s, dev);
  }
  e = cudaFreeAsync(ws, s);
  if (st == LVB_OK && e != cudaSuccess) return fail_cuda(e, op, "workspace free");
  return st;
}

}  // extern "C"
