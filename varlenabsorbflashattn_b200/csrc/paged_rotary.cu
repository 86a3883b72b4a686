// Rotation of packed queries and keys by their positions, and the append of new keys and values to a paged cache with that
// rotation on the way.
//
// A pair (x1, x2) of a head at position p turns by the angle p * w_i, whose cosine and sine come from a table:
//   y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin      (back, which is the gradient: the same with -sin).
// Every value is read once and written once, so HBM bounds the kernel.  A thread owns the same `VW` pairs of several heads of one
// token: the cosines and sines (twice the bytes of a head's 16-bit pairs) are read once per thread instead of once per head, and
// the loads of four heads are in flight together.  Arithmetic is fp32, one rounding at the end.
#include "paged_kernels.cuh"
#include "profile.cuh"

namespace vafa {
namespace {

struct HeadGroup {
  const void* src;
  void* dst;                              // packed output, or the cache
  int64_t token_stride, head_stride;      // of src
  int64_t page_stride, slot_stride, dst_head_stride;
  int first;                              // index of its first head among all groups' heads
  int rotate;
  int cached;                             // dst is a cache: the token's page and slot give the place
};

struct RotaryParams {
  HeadGroup g[3];
  int n_groups, heads;                    // heads of all groups
  const float* cos;
  const float* sin;
  const int32_t* positions;
  const int32_t* cu;
  const int32_t* lens;                    // append only
  const int32_t* table;
  int64_t table_stride;
  int n_seg, total, D, R, table_rows, num_pages, page_size, max_pages;
  int chunks, lanes, tokens_per_block;    // chunks of a head, head lanes, tokens of a block
  float sign;
  int32_t* status;
};

template <typename T, int N> struct alignas(sizeof(T) * N) Vec { T v[N]; };
template <int N> struct alignas(N * 4 > 16 ? 16 : N * 4) Floats { float v[N]; };

// What becomes of a token.
enum Fate { kDone = 0, kZeros = 1, kNaNs = 2 };

template <typename T, int VW, bool INTER, bool APPEND>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryParams p) {
  const int per_token = p.chunks * p.lanes;
  const int slot_in_block = threadIdx.x / per_token;
  const int64_t t64 = (int64_t)blockIdx.x * p.tokens_per_block + slot_in_block;
  if (slot_in_block >= p.tokens_per_block || t64 >= p.total) return;
  const int t = (int)t64;
  const int in_token = threadIdx.x - slot_in_block * per_token;
  const int lane = in_token / p.chunks, c = in_token - lane * p.chunks;

  int fate = kDone;
  int pos = 0, page = 0, slot = 0;
  if constexpr (APPEND) {
    int seq = t;
    int behind = 1;                       // tokens from this one to the end of its sequence, itself among them
    if (p.cu != nullptr) {
      seq = find_segment(p.cu, p.n_seg, t);
      behind = p.cu[seq + 1] - t;
    }
    if (behind < 1) {
      fate = kZeros;                      // behind the last sequence
    } else {
      const int len = p.lens[seq];
      pos = len - behind;
      const int row = pos / p.page_size;
      if (len == 0) {
        fate = kZeros;                    // a padding sequence
      } else if (pos < 0 || row >= p.max_pages || (p.cos != nullptr && pos >= p.table_rows)) {
        fate = kNaNs;
      } else {
        page = p.table[seq * p.table_stride + row];
        slot = pos - row * p.page_size;
        if (page < 0 || page >= p.num_pages) fate = kNaNs;
      }
      if (fate == kNaNs && in_token == 0) report_error(p.status, kBadCacheIndex, kSiteAppend, t);
    }
  } else {
    if (p.positions != nullptr) {
      pos = p.positions[t];
    } else {
      const int seg = find_segment(p.cu, p.n_seg, t);
      pos = t - p.cu[seg];
      if (t >= p.cu[p.n_seg]) fate = kZeros;
    }
    if (fate == kDone && (pos < 0 || pos >= p.table_rows)) {
      fate = kNaNs;
      if (in_token == 0) report_error(p.status, kBadCacheIndex, kSiteRotary, t);
    }
  }

  const bool turned = c * 2 * VW < p.R;   // a chunk of the dims that rotate, or of those that pass through
  float cs[VW], sn[VW];
  if (turned && fate == kDone && p.cos != nullptr) {
    const int64_t at = (int64_t)pos * (p.R / 2) + c * VW;
    constexpr int N = VW > 4 ? 4 : VW;
#pragma unroll
    for (int j = 0; j < VW; j += N) {
      const Floats<N> a = *reinterpret_cast<const Floats<N>*>(p.cos + at + j);
      const Floats<N> b = *reinterpret_cast<const Floats<N>*>(p.sin + at + j);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        cs[j + e] = a.v[e];
        sn[j + e] = p.sign * b.v[e];
      }
    }
  }
  // the two vectors of a chunk: both halves of its pairs, or 2 VW neighbours
  const int d0 = turned && !INTER ? c * VW : 2 * c * VW;
  const int d1 = turned && !INTER ? p.R / 2 + c * VW : d0 + VW;

  constexpr int kBatch = 4;
  using V = Vec<T, VW>;
  for (int h0 = lane; h0 < p.heads; h0 += kBatch * p.lanes) {
    V x[kBatch], y[kBatch];
    T* out[kBatch];
    bool rot[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int h = h0 + b * p.lanes;
      out[b] = nullptr;
      rot[b] = false;
      if (h < p.heads) {
        int gi = 0;
        if (p.n_groups > 1 && h >= p.g[1].first) gi = 1;
        if (p.n_groups > 2 && h >= p.g[2].first) gi = 2;
        const HeadGroup& g = p.g[gi];
        const int hg = h - g.first;
        rot[b] = g.rotate && turned;
        if (!g.cached || fate == kDone) {
          out[b] = reinterpret_cast<T*>(g.dst) + hg * g.dst_head_stride +
                   (g.cached ? page * g.page_stride + slot * g.slot_stride : (int64_t)t * g.page_stride);
          if (fate == kDone) {
            const T* src = reinterpret_cast<const T*>(g.src) + (int64_t)t * g.token_stride + hg * g.head_stride;
            x[b] = *reinterpret_cast<const V*>(src + d0);
            y[b] = *reinterpret_cast<const V*>(src + d1);
          }
        }
      }
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (out[b] == nullptr) continue;
      if (fate != kDone) {
        const T fill = from_float<T>(fate == kZeros ? 0.f : __int_as_float(0x7fc00000));
#pragma unroll
        for (int j = 0; j < VW; ++j) x[b].v[j] = y[b].v[j] = fill;
      } else if (rot[b]) {
        if constexpr (INTER) {
          V u, w;
#pragma unroll
          for (int j = 0; j < VW; ++j) {
            const T a = 2 * j < VW ? x[b].v[(2 * j) % VW] : y[b].v[(2 * j) % VW];
            const T e = 2 * j + 1 < VW ? x[b].v[(2 * j + 1) % VW] : y[b].v[(2 * j + 1) % VW];
            const float f = to_float(a), g = to_float(e);
            const T r0 = from_float<T>(f * cs[j] - g * sn[j]), r1 = from_float<T>(g * cs[j] + f * sn[j]);
            if (2 * j < VW) u.v[(2 * j) % VW] = r0; else w.v[(2 * j) % VW] = r0;
            if (2 * j + 1 < VW) u.v[(2 * j + 1) % VW] = r1; else w.v[(2 * j + 1) % VW] = r1;
          }
          x[b] = u;
          y[b] = w;
        } else {
#pragma unroll
          for (int j = 0; j < VW; ++j) {
            const float f = to_float(x[b].v[j]), g = to_float(y[b].v[j]);
            x[b].v[j] = from_float<T>(f * cs[j] - g * sn[j]);
            y[b].v[j] = from_float<T>(g * cs[j] + f * sn[j]);
          }
        }
      }
      *reinterpret_cast<V*>(out[b] + d0) = x[b];
      *reinterpret_cast<V*>(out[b] + d1) = y[b];
    }
  }
}

template <typename T, int VW>
void launch(const RotaryParams& p, bool inter, bool append, unsigned blocks, int threads, cudaStream_t s) {
  if (append) {
    if (inter) rotary_kernel<T, VW, true, true><<<blocks, threads, 0, s>>>(p);
    else rotary_kernel<T, VW, false, true><<<blocks, threads, 0, s>>>(p);
  } else {
    if (inter) rotary_kernel<T, VW, true, false><<<blocks, threads, 0, s>>>(p);
    else rotary_kernel<T, VW, false, false><<<blocks, threads, 0, s>>>(p);
  }
}

template <typename T>
void launch_by_width(int vw, const RotaryParams& p, bool inter, bool append, unsigned blocks, int threads, cudaStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (vw == 8) return launch<T, 8>(p, inter, append, blocks, threads, s);
  }
  if (vw == 4) return launch<T, 4>(p, inter, append, blocks, threads, s);
  if (vw == 2) return launch<T, 2>(p, inter, append, blocks, threads, s);
  launch<T, 1>(p, inter, append, blocks, threads, s);
}

// Elements of a vector: the widest that divides the rotating half and that every address is a multiple of.
int vector_width(const RotaryParams& p, int es) {
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

// Heads of a thread: four where that leaves every SM with enough threads, fewer for small batches.
int launch_rotary(RotaryParams& p, int heads, int dtype, bool inter, bool append, int kernel_id, cudaStream_t s) {
  const int vw = vector_width(p, elem_size(dtype));
  p.heads = heads;
  p.chunks = p.D / (2 * vw);
  if (p.total == 0 || heads == 0) return 0;
  const long long threads = (long long)p.total * p.chunks * heads;
  const long long each = threads / (148 * 1024);
  const int per_thread = each < 1 ? 1 : each > 4 ? 4 : (int)each;
  const int most = 256 / p.chunks;
  const int want = (heads + per_thread - 1) / per_thread;
  p.lanes = want < most ? want : most;
  p.tokens_per_block = 256 / (p.chunks * p.lanes);
  const unsigned blocks = (unsigned)(((long long)p.total + p.tokens_per_block - 1) / p.tokens_per_block);
  const int block = p.tokens_per_block * p.chunks * p.lanes;
  LaunchScope scope(kernel_id, s);
  if (dtype == VAFA_F32) launch_by_width<float>(vw, p, inter, append, blocks, block, s);
  else if (dtype == VAFA_BF16) launch_by_width<__nv_bfloat16>(vw, p, inter, append, blocks, block, s);
  else launch_by_width<__half>(vw, p, inter, append, blocks, block, s);
  VAFA_LAUNCH_CHECK(append ? "paged_append_kernel" : "rotary_kernel");
  return 0;
}

}  // namespace

int rotary_launch(const vafa_rotary_args* a, cudaStream_t s) {
  RotaryParams p{};
  const int64_t D = a->head_dim;
  int heads = 0;
  auto add = [&](const void* src, void* dst, int64_t ts, int64_t hs, int n) {
    if (n == 0) return;
    // a packed output has one "page" per token
    p.g[p.n_groups++] = HeadGroup{src, dst, of(a->total, ts), of(n, hs), n * D, 0, D, heads, 1, 0};
    heads += n;
  };
  add(a->q, a->q_out, a->q_token_stride, a->q_head_stride, a->num_heads);
  add(a->k, a->k_out, a->k_token_stride, a->k_head_stride, a->num_kv_heads);
  p.cos = a->cos; p.sin = a->sin; p.positions = a->positions; p.cu = a->cu_seqlens;
  p.n_seg = a->n_seg; p.total = a->total; p.D = a->head_dim; p.R = a->rotary_dim; p.table_rows = a->table_rows;
  p.sign = a->inverse ? -1.f : 1.f;
  p.status = a->status;
  return launch_rotary(p, heads, a->dtype, a->interleaved != 0, false, kKRotary, s);
}

int paged_append_launch(const vafa_paged_append_args* a, cudaStream_t s) {
  RotaryParams p{};
  const int64_t D = a->head_dim;
  const int rotate = a->cos != nullptr;
  int heads = 0;
  if (a->q != nullptr) {
    p.g[p.n_groups++] = HeadGroup{a->q, a->q_out, of(a->total, a->q_token_stride), of(a->num_heads, a->q_head_stride), a->num_heads * D, 0, D, heads, rotate, 0};
    heads += a->num_heads;
  }
  p.g[p.n_groups++] = HeadGroup{a->k, a->k_cache, of(a->total, a->k_token_stride), of(a->num_kv_heads, a->k_head_stride),
                                of(a->num_pages, a->k_page_stride), of(a->page_size, a->k_slot_stride), of(a->num_kv_heads, a->k_cache_head_stride), heads, rotate, 1};
  heads += a->num_kv_heads;
  p.g[p.n_groups++] = HeadGroup{a->v, a->v_cache, of(a->total, a->v_token_stride), of(a->num_kv_heads, a->v_head_stride),
                                of(a->num_pages, a->v_page_stride), of(a->page_size, a->v_slot_stride), of(a->num_kv_heads, a->v_cache_head_stride), heads, 0, 1};
  heads += a->num_kv_heads;
  p.cos = a->cos; p.sin = a->sin; p.cu = a->cu_seqlens; p.lens = a->cache_seqlens; p.table = a->page_table;
  p.table_stride = a->table_stride;
  p.n_seg = a->n_seq; p.total = a->total; p.D = a->head_dim; p.R = rotate ? a->rotary_dim : 0; p.table_rows = a->table_rows;
  p.num_pages = a->num_pages; p.page_size = a->page_size; p.max_pages = a->max_pages;
  p.sign = 1.f;
  p.status = a->status;
  return launch_rotary(p, heads, a->dtype, a->interleaved != 0, true, kKPagedAppend, s);
}

}  // namespace vafa
