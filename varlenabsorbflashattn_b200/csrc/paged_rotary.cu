// Rotation of packed queries and keys by their positions, and the append of new keys and values to a paged cache with that
// rotation on the way.
//
// A pair (x1, x2) of a head at position p turns by the angle p * w_i, whose cosine and sine come from a table:
//   y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin      (back, which is the gradient: the same with -sin).
// Every value is read once and written once, so HBM bounds a long batch; those go through shared memory (paged_rotary_rows.cu).  The
// kernel here does the others, where latency counts: a thread owns the same VW pairs of up to two heads of a token, reads them
// before it looks up the position and the angles (the chain segment - position - angle costs as much as the values), and
// reads the cosines and sines, twice the bytes of a head's 16-bit pairs, once for both.  Arithmetic is fp32, one rounding at the end.
#include "paged_rotary.cuh"

namespace vafa {
namespace rotary {
namespace {

constexpr int kHeads = 2;  // heads of a thread

struct Shape {
  int chunks, lanes, passes;   // chunks of a head, head lanes of a token, groups of kHeads x lanes heads
  int tokens_per_block;
};

template <typename T, int VW, bool INTER, bool APPEND>
__global__ void __launch_bounds__(256) rotary_kernel(const Params p, const Shape w) {
  const int per_token = w.chunks * w.lanes;
  const int in_block = threadIdx.x / per_token;
  const int in_token = threadIdx.x - in_block * per_token;
  const int lane = in_token / w.chunks, c = in_token - lane * w.chunks;
  const int64_t t64 = (int64_t)blockIdx.x * w.tokens_per_block + in_block;
  if (in_block >= w.tokens_per_block || t64 >= p.total) return;
  const int t = (int)t64;
  const bool turned = c * 2 * VW < p.R;   // a chunk of the dims that rotate, or of those that pass through
  // the two vectors of a chunk: both halves of its pairs, or 2 VW neighbours
  const int d0 = turned && !INTER ? c * VW : 2 * c * VW;
  const int d1 = turned && !INTER ? p.R / 2 + c * VW : d0 + VW;
  // a field of the head's group, by selects (the parameters are not indexed)
  auto of_group = [&](int h, auto field) { return h >= p.g[2].first ? field(p.g[2]) : h >= p.g[1].first ? field(p.g[1]) : field(p.g[0]); };

  Vec<T, VW> x[kHeads], y[kHeads];
  auto load = [&](int pass) {
#pragma unroll
    for (int b = 0; b < kHeads; ++b) {
      const int h = (pass * kHeads + b) * w.lanes + lane;
      if (h < p.heads) {
        const T* src = reinterpret_cast<const T*>(of_group(h, [](const HeadGroup& g) { return g.src; })) +
                       (int64_t)t * of_group(h, [](const HeadGroup& g) { return g.token_stride; }) +
                       (h - of_group(h, [](const HeadGroup& g) { return g.first; })) * of_group(h, [](const HeadGroup& g) { return g.head_stride; });
        x[b] = *reinterpret_cast<const Vec<T, VW>*>(src + d0);
        y[b] = *reinterpret_cast<const Vec<T, VW>*>(src + d1);
      }
    }
  };
  load(0);
  int pos, page, slot;
  const Fate fate = place_of<APPEND>(p, t, in_token == 0, &pos, &page, &slot);
  float cs[VW], sn[VW];
  if (turned && fate == kDone && p.cos != nullptr) {
    const int64_t at = (int64_t)pos * (p.R / 2) + c * VW;
    load_angles<VW>(p.cos + at, p.sin + at, p.sign, cs, sn);
  }
  for (int pass = 0; pass < w.passes; ++pass) {
    if (pass > 0) load(pass);
#pragma unroll
    for (int b = 0; b < kHeads; ++b) {
      const int h = (pass * kHeads + b) * w.lanes + lane;
      if (h >= p.heads) break;
      const bool cached = APPEND && of_group(h, [](const HeadGroup& g) { return g.cached; });
      const bool turns = turned && (!APPEND || of_group(h, [](const HeadGroup& g) { return g.rotate; }));
      if (cached && fate != kDone) continue;
      const int64_t page_stride = of_group(h, [](const HeadGroup& g) { return g.page_stride; });
      T* const out = reinterpret_cast<T*>(of_group(h, [](const HeadGroup& g) { return g.dst; })) +
                     (h - of_group(h, [](const HeadGroup& g) { return g.first; })) * of_group(h, [](const HeadGroup& g) { return g.dst_head_stride; }) +
                     (cached ? page * page_stride + slot * of_group(h, [](const HeadGroup& g) { return g.slot_stride; }) : t * page_stride);
      if (fate != kDone) {
        const T fill = from_float<T>(fate == kZeros ? 0.f : __int_as_float(0x7fc00000));
#pragma unroll
        for (int j = 0; j < VW; ++j) x[b].v[j] = y[b].v[j] = fill;
      } else if (turns) {
        rotate<T, VW, INTER>(x[b], y[b], cs, sn);
      }
      *reinterpret_cast<Vec<T, VW>*>(out + d0) = x[b];
      *reinterpret_cast<Vec<T, VW>*>(out + d1) = y[b];
    }
  }
}

template <typename T, int VW>
void launch(const Params& p, const Shape& w, bool inter, bool append, unsigned blocks, int threads, cudaStream_t s) {
  if (append) {
    if (inter) rotary_kernel<T, VW, true, true><<<blocks, threads, 0, s>>>(p, w);
    else rotary_kernel<T, VW, false, true><<<blocks, threads, 0, s>>>(p, w);
  } else {
    if (inter) rotary_kernel<T, VW, true, false><<<blocks, threads, 0, s>>>(p, w);
    else rotary_kernel<T, VW, false, false><<<blocks, threads, 0, s>>>(p, w);
  }
}

template <typename T>
void launch_by_width(int vw, const Params& p, const Shape& w, bool inter, bool append, unsigned blocks, int threads, cudaStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (vw == 8) return launch<T, 8>(p, w, inter, append, blocks, threads, s);
  }
  if (vw == 4) return launch<T, 4>(p, w, inter, append, blocks, threads, s);
  if (vw == 2) return launch<T, 2>(p, w, inter, append, blocks, threads, s);
  launch<T, 1>(p, w, inter, append, blocks, threads, s);
}

// Elements of a vector: the widest that divides the rotating half and that every address is a multiple of.
int vector_width(const Params& p, int es) {
  auto fits = [&](int w) {
    if (p.R > 0 && ((p.R / 2) % w || ((uintptr_t)p.cos | (uintptr_t)p.sin) % (w * 4 < 16 ? w * 4 : 16))) return false;
    for (int i = 0; i < p.n_groups; ++i) {
      const HeadGroup& g = p.g[i];
      if (((uintptr_t)g.src | (uintptr_t)g.dst) % (w * es)) return false;
      if ((g.token_stride | g.head_stride | g.page_stride | g.slot_stride | g.dst_head_stride) % w) return false;
    }
    return true;
  };
  int w = 16 / es;
  while (w > 1 && !fits(w)) w >>= 1;
  return w;
}

// The stride of a dim, which says nothing where the dim has one element.
int64_t of(int n, int64_t stride) { return n > 1 ? stride : 0; }

int launch_rotary(Params& p, int heads, int dtype, bool inter, bool append, int kernel_id, cudaStream_t s) {
  const int vw = vector_width(p, elem_size(dtype));
  p.heads = heads;
  for (int i = p.n_groups; i < 3; ++i) p.g[i].first = 0x7fffffff;
  if (p.total == 0 || heads == 0) return 0;
  const int rc = launch_rows(p, vw, dtype, inter, append, s);
  if (rc <= 0) return rc;
  // Two heads a thread, one where threads are few: one | two heads, 256 new tokens of 48 heads of 128 3.9 | 4.2 us, 400 tokens of 40 heads
  // 5.3 | 3.9, 800 tokens 7.5 | 6.0.
  Shape w;
  w.chunks = p.D / (2 * vw);
  const int most = 256 / w.chunks;
  const bool few = (long long)p.total * w.chunks * heads < 148LL * 768;
  const int want = few ? heads : (heads + kHeads - 1) / kHeads;
  w.lanes = want < most ? want : most;
  w.passes = (heads + kHeads * w.lanes - 1) / (kHeads * w.lanes);
  w.tokens_per_block = 256 / (w.chunks * w.lanes);
  const unsigned blocks = (unsigned)(((long long)p.total + w.tokens_per_block - 1) / w.tokens_per_block);
  const int block = w.tokens_per_block * w.chunks * w.lanes;
  LaunchScope scope(kernel_id, s);
  if (dtype == VAFA_F32) launch_by_width<float>(vw, p, w, inter, append, blocks, block, s);
  else if (dtype == VAFA_BF16) launch_by_width<__nv_bfloat16>(vw, p, w, inter, append, blocks, block, s);
  else launch_by_width<__half>(vw, p, w, inter, append, blocks, block, s);
  VAFA_LAUNCH_CHECK(append ? "paged_append_kernel" : "rotary_kernel");
  return 0;
}

}  // namespace
}  // namespace rotary

int rotary_launch(const vafa_rotary_args* a, cudaStream_t s) {
  rotary::Params p{};
  const int64_t D = a->head_dim;
  int heads = 0;
  auto add = [&](const void* src, void* dst, int64_t ts, int64_t hs, int n) {
    if (n == 0) return;
    // a packed output has one "page" per token
    p.g[p.n_groups++] = rotary::HeadGroup{src, dst, rotary::of(a->total, ts), rotary::of(n, hs), n * D, 0, D, heads, 1, 0};
    heads += n;
  };
  add(a->q, a->q_out, a->q_token_stride, a->q_head_stride, a->num_heads);
  add(a->k, a->k_out, a->k_token_stride, a->k_head_stride, a->num_kv_heads);
  p.cos = a->cos; p.sin = a->sin; p.positions = a->positions; p.cu = a->cu_seqlens;
  p.n_seg = a->n_seg; p.total = a->total; p.D = a->head_dim; p.R = a->rotary_dim; p.table_rows = a->table_rows;
  p.sign = a->inverse ? -1.f : 1.f;
  p.status = a->status;
  return rotary::launch_rotary(p, heads, a->dtype, a->interleaved != 0, false, kKRotary, s);
}

int paged_append_launch(const vafa_paged_append_args* a, cudaStream_t s) {
  rotary::Params p{};
  const int64_t D = a->head_dim;
  const int rotate = a->cos != nullptr;
  int heads = 0;
  if (a->q != nullptr) {
    p.g[p.n_groups++] = rotary::HeadGroup{a->q, a->q_out, rotary::of(a->total, a->q_token_stride), rotary::of(a->num_heads, a->q_head_stride), a->num_heads * D, 0, D, heads, rotate, 0};
    heads += a->num_heads;
  }
  p.g[p.n_groups++] = rotary::HeadGroup{a->k, a->k_cache, rotary::of(a->total, a->k_token_stride), rotary::of(a->num_kv_heads, a->k_head_stride),
                                rotary::of(a->num_pages, a->k_page_stride), rotary::of(a->page_size, a->k_slot_stride), rotary::of(a->num_kv_heads, a->k_cache_head_stride), heads, rotate, 1};
  heads += a->num_kv_heads;
  p.g[p.n_groups++] = rotary::HeadGroup{a->v, a->v_cache, rotary::of(a->total, a->v_token_stride), rotary::of(a->num_kv_heads, a->v_head_stride),
                                rotary::of(a->num_pages, a->v_page_stride), rotary::of(a->page_size, a->v_slot_stride), rotary::of(a->num_kv_heads, a->v_cache_head_stride), heads, 0, 1};
  heads += a->num_kv_heads;
  p.cos = a->cos; p.sin = a->sin; p.cu = a->cu_seqlens; p.lens = a->cache_seqlens; p.table = a->page_table;
  p.table_stride = a->table_stride;
  p.n_seg = a->n_seq; p.total = a->total; p.D = a->head_dim; p.R = rotate ? a->rotary_dim : 0; p.table_rows = a->table_rows;
  p.num_pages = a->num_pages; p.page_size = a->page_size; p.max_pages = a->max_pages;
  p.sign = 1.f;
  p.status = a->status;
  return rotary::launch_rotary(p, heads, a->dtype, a->interleaved != 0, true, kKPagedAppend, s);
}

}  // namespace vafa
