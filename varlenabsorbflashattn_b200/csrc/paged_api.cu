// C ABI of the rotation, the paged append and the paged decode: argument checks and the choice of a decode tile.
#include <string.h>

#include <initializer_list>

#include "paged_decode.cuh"

namespace vafa {
namespace {

bool dtype_ok(int d) { return d == VAFA_F32 || d == VAFA_BF16 || d == VAFA_F16; }
bool dim_ok(int d) { return d == 16 || d == 32 || d == 64 || d == 128 || d == 256; }
bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Addresses of whole elements, and of whole 32-bit words.
int check_addresses(int dtype, std::initializer_list<const void*> tensors, std::initializer_list<const void*> words) {
  for (const void* p : tensors)
    if (!aligned(p, elem_size(dtype))) return fail(VAFA_ERR_INVALID, "tensors must be aligned to their elements");
  for (const void* p : words)
    if (!aligned(p, 4)) return fail(VAFA_ERR_INVALID, "positions, lengths, tables, lse and status must be 4-byte aligned");
  return 0;
}

// Heads of a call of the rotation and the append, which count them in 32 bits.
int check_heads(long long heads) { return heads > (1 << 30) ? fail(VAFA_ERR_UNSUPPORTED, "%lld heads", heads) : 0; }

int check_table(const float* cos, const float* sin, int R, int D, int rows) {
  if (!cos || !sin) return fail(VAFA_ERR_INVALID, "null cos/sin");
  if (!aligned(cos, 4) || !aligned(sin, 4)) return fail(VAFA_ERR_INVALID, "cos/sin must be 4-byte aligned");
  if (R < 2 || R > D || (R & 1)) return fail(VAFA_ERR_INVALID, "rotary_dim %d must be even, 2 to head_dim %d", R, D);
  if (rows < 0) return fail(VAFA_ERR_INVALID, "bad table_rows %d", rows);
  return 0;
}

int check_pointers(const void* k, const void* v, const int32_t* lens, const int32_t* table) {
  if (!k || !v) return fail(VAFA_ERR_INVALID, "null cache");
  if (!lens || !table) return fail(VAFA_ERR_INVALID, "null cache_seqlens/page_table");
  return 0;
}

int check_cache(int n_seq, int pages, int page_size, int max_pages) {
  if (n_seq < 1 || pages < 1 || page_size < 1 || max_pages < 1)
    return fail(VAFA_ERR_INVALID, "bad sizes n_seq=%d num_pages=%d page_size=%d max_pages=%d", n_seq, pages, page_size, max_pages);
  if ((long long)max_pages * page_size > 0x7fffffffLL - 65536)
    return fail(VAFA_ERR_INVALID, "max_pages %d x page_size %d exceeds int32 range", max_pages, page_size);
  return 0;
}

int check_decode(const vafa_paged_attn_args* a) {
  if (!a) return fail(VAFA_ERR_INVALID, "null args");
  if (!dtype_ok(a->dtype)) return fail(VAFA_ERR_INVALID, "bad dtype %d", a->dtype);
  if (!dim_ok(a->head_dim)) return fail(VAFA_ERR_UNSUPPORTED, "head_dim %d not supported (16/32/64/128/256)", a->head_dim);
  if (a->q_len < 1 || a->num_heads < 1 || a->num_kv_heads < 1 || a->num_heads % a->num_kv_heads)
    return fail(VAFA_ERR_INVALID, "bad sizes q_len=%d H=%d H_kv=%d (H_kv must divide H)", a->q_len, a->num_heads, a->num_kv_heads);
  if ((long long)a->q_len * a->num_heads > (1 << 18) || a->num_kv_heads > 0xffff) return fail(VAFA_ERR_UNSUPPORTED, "q_len %d x %d heads", a->q_len, a->num_heads);
  if (a->n_seq > (1 << 30)) return fail(VAFA_ERR_UNSUPPORTED, "n_seq %d", a->n_seq);  // (a CTA's threads share out the sequences in 32 bits)
  return check_cache(a->n_seq, a->num_pages, a->page_size, a->max_pages);
}

paged::Plan plan_for(const vafa_paged_attn_args* a) {
  const int R = a->q_len * (a->num_heads / a->num_kv_heads);
  return a->dtype == VAFA_F32 ? paged::plan_f32(a->head_dim, R) : a->dtype == VAFA_BF16 ? paged::plan_bf16(a->head_dim, R) : paged::plan_f16(a->head_dim, R);
}

// CTAs of a call, and whether a unit can end up in several of them: from the room that the page table has, as the lengths are on the device.
struct Cut {
  int ctas;
  bool splits;
  size_t part_o, part_ml, meta;
};

int cut_for(const vafa_paged_attn_args* a, const paged::Plan& plan, Cut* c) {
  int sms = a->sm_count;
  if (sms <= 0) {
    int dev = 0;
    VAFA_CUDA_CHECK(cudaGetDevice(&dev));
    VAFA_CUDA_CHECK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  }
  const long long per_unit = ((long long)a->max_pages * a->page_size + plan.bk - 1) / plan.bk;
  const long long units = (long long)a->num_kv_heads * plan.row_tiles;
  if (units * (per_unit + paged::kUnitCost) > 0x7fffffffLL) return fail(VAFA_ERR_UNSUPPORTED, "a sequence has too many heads and keys");
  const long long most = units * per_unit * a->n_seq;
  // a CTA for every block until the SMs are full (pieces of at least 1 | 2 | 4 | 8 slots, one cache of 512 keys: 8.6 | 9.6 | 11.3 | 13.9 us)
  c->ctas = (int)(most < (long long)sms * plan.ctas_per_sm ? most : (long long)sms * plan.ctas_per_sm);
  c->splits = per_unit > 1;
  c->part_o = align_up((size_t)2 * c->ctas * plan.rows * a->head_dim * 4, 256);
  c->part_ml = align_up((size_t)2 * c->ctas * plan.rows * 8, 256);
  c->meta = align_up((size_t)c->ctas * 16, 256);
  return 0;
}

}  // namespace

size_t paged_decode_workspace(const vafa_paged_attn_args* a) {
  Cut c;
  if (cut_for(a, plan_for(a), &c)) return 0;
  return c.part_o + c.part_ml + c.meta;
}

int paged_decode_launch(const vafa_paged_attn_args* a, cudaStream_t s) {
  const paged::Plan plan = plan_for(a);
  Cut c;
  if (const int rc = cut_for(a, plan, &c)) return rc;
  const size_t need = c.part_o + c.part_ml + c.meta;
  if (!a->workspace || a->workspace_bytes < need) return fail(VAFA_ERR_WORKSPACE, "workspace too small: have %zu, need %zu", a->workspace_bytes, need);
  if (!aligned(a->workspace, 256)) return fail(VAFA_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  paged::DecodeParams p;
  memset(&p, 0, sizeof(p));
  p.q = a->q; p.k = a->k_cache; p.v = a->v_cache; p.o = a->o; p.lse = a->lse;
  p.lens = a->cache_seqlens; p.table = a->page_table;
  p.q_seq = a->q_seq_stride; p.q_token = a->q_token_stride; p.q_head = a->q_head_stride;
  p.k_page = a->k_page_stride; p.k_slot = a->k_slot_stride; p.k_head = a->k_cache_head_stride;
  p.v_page = a->v_page_stride; p.v_slot = a->v_slot_stride; p.v_head = a->v_cache_head_stride;
  p.table_stride = a->table_stride;
  p.n_seq = a->n_seq; p.T = a->q_len; p.H = a->num_heads; p.H_kv = a->num_kv_heads;
  p.g = a->num_heads / a->num_kv_heads; p.R = p.T * p.g;
  p.row_tiles = plan.row_tiles; p.num_pages = a->num_pages; p.page_size = a->page_size;
  // j / page_size by a product: page_mul = ceil(2^(32 + shift) / page_size) with 2^shift < page_size <= 2^(shift + 1) is off by less
  // than page_size / 2^(32 + shift) <= 2^-31 of j, which stays below 1 / page_size of a step for j < 2^31
  int shift = 0;
  while ((1ll << (shift + 1)) <= a->page_size) ++shift;
  p.page_shift = shift;
  p.page_mul = (a->page_size & (a->page_size - 1)) == 0 ? 0 : (uint32_t)(((1ull << (32 + shift)) + a->page_size - 1) / a->page_size);
  p.capacity = a->max_pages * a->page_size;
  p.scale_log2 = a->scale * kLog2e;
  char* ws = (char*)a->workspace;
  p.part_o = (float*)ws;
  p.part_ml = (float2*)(ws + c.part_o);
  p.meta = (int4*)(ws + c.part_o + c.part_ml);
  p.status = a->status;
  return plan.launch(p, c.ctas, c.splits, s);
}

}  // namespace vafa

using namespace vafa;

extern "C" {
#pragma GCC visibility push(default)

int vafa_rotary(const vafa_rotary_args* a, vafa_stream_t stream) {
  if (!a) return fail(VAFA_ERR_INVALID, "null args");
  if (!dtype_ok(a->dtype)) return fail(VAFA_ERR_INVALID, "bad dtype %d", a->dtype);
  if (!dim_ok(a->head_dim)) return fail(VAFA_ERR_UNSUPPORTED, "head_dim %d not supported (16/32/64/128/256)", a->head_dim);
  if (a->total < 0 || a->num_heads < 0 || a->num_kv_heads < 0) return fail(VAFA_ERR_INVALID, "bad sizes");
  if (const int rc = check_table(a->cos, a->sin, a->rotary_dim, a->head_dim, a->table_rows)) return rc;
  if (!a->positions && (!a->cu_seqlens || a->n_seg < 1)) return fail(VAFA_ERR_INVALID, "neither positions nor cu_seqlens");
  if (a->total > 0 && ((a->num_heads > 0 && (!a->q || !a->q_out)) || (a->num_kv_heads > 0 && (!a->k || !a->k_out))))
    return fail(VAFA_ERR_INVALID, "null q/k");
  if (const int rc = check_heads((long long)a->num_heads + a->num_kv_heads)) return rc;
  if (const int rc = check_addresses(a->dtype, {a->q, a->k, a->q_out, a->k_out}, {a->positions, a->cu_seqlens, a->status})) return rc;
  return rotary_launch(a, (cudaStream_t)stream);
}

int vafa_paged_append(const vafa_paged_append_args* a, vafa_stream_t stream) {
  if (!a) return fail(VAFA_ERR_INVALID, "null args");
  if (!dtype_ok(a->dtype)) return fail(VAFA_ERR_INVALID, "bad dtype %d", a->dtype);
  if (!dim_ok(a->head_dim)) return fail(VAFA_ERR_UNSUPPORTED, "head_dim %d not supported (16/32/64/128/256)", a->head_dim);
  if (a->total < 0 || a->num_kv_heads < 1 || (a->q && a->num_heads < 1)) return fail(VAFA_ERR_INVALID, "bad sizes");
  int rc;
  if (a->cos || a->sin) {
    if ((rc = check_table(a->cos, a->sin, a->rotary_dim, a->head_dim, a->table_rows))) return rc;
  } else if (a->q) {
    return fail(VAFA_ERR_INVALID, "q without cos/sin");
  }
  if ((rc = check_pointers(a->k_cache, a->v_cache, a->cache_seqlens, a->page_table))) return rc;
  if ((rc = check_cache(a->n_seq, a->num_pages, a->page_size, a->max_pages))) return rc;
  if (!a->cu_seqlens && a->total != a->n_seq) return fail(VAFA_ERR_INVALID, "without cu_seqlens total %d must be n_seq %d", a->total, a->n_seq);
  if (a->total > 0 && (!a->k || !a->v || (a->q && !a->q_out))) return fail(VAFA_ERR_INVALID, "null k/v/q_out");
  if ((rc = check_heads((a->q ? a->num_heads : 0) + 2LL * a->num_kv_heads))) return rc;
  if ((rc = check_addresses(a->dtype, {a->q, a->k, a->v, a->q_out, a->k_cache, a->v_cache}, {a->cu_seqlens, a->cache_seqlens, a->page_table, a->status})))
    return rc;
  return paged_append_launch(a, (cudaStream_t)stream);
}

size_t vafa_paged_decode_workspace_bytes(const vafa_paged_attn_args* a) {
  return check_decode(a) ? 0 : paged_decode_workspace(a);
}

int vafa_paged_decode(const vafa_paged_attn_args* a, vafa_stream_t stream) {
  if (const int rc = check_decode(a)) return rc;
  if (!a->q || !a->o) return fail(VAFA_ERR_INVALID, "null q/o");
  if (const int rc = check_pointers(a->k_cache, a->v_cache, a->cache_seqlens, a->page_table)) return rc;
  const int es = elem_size(a->dtype);
  auto of = [](int n, int64_t stride) { return n > 1 ? stride : 0; };  // (a dim of one element may have any stride)
  const int64_t strides = of(a->n_seq, a->q_seq_stride) | of(a->q_len, a->q_token_stride) | of(a->num_heads, a->q_head_stride) |
                          of(a->num_pages, a->k_page_stride | a->v_page_stride) | of(a->page_size, a->k_slot_stride | a->v_slot_stride) |
                          of(a->num_kv_heads, a->k_cache_head_stride | a->v_cache_head_stride);
  if (!aligned(a->q, 16) || !aligned(a->k_cache, 16) || !aligned(a->v_cache, 16) || !aligned(a->o, 16) || (strides * es) % 16)
    return fail(VAFA_ERR_INVALID, "q, o and the caches need 16-byte aligned bases and strides");
  if (const int rc = check_addresses(a->dtype, {}, {a->cache_seqlens, a->page_table, a->lse, a->status})) return rc;
  return paged_decode_launch(a, (cudaStream_t)stream);
}

#pragma GCC visibility pop
}
