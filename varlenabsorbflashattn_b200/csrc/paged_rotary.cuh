// What the two rotation kernels share: the work of a call, and where a token stands.
#pragma once
#include "paged_kernels.cuh"
#include "profile.cuh"

namespace vafa {
namespace rotary {

struct HeadGroup {
  const void* src;
  void* dst;                              // packed output, or the cache
  int64_t token_stride, head_stride;      // of src
  int64_t page_stride, slot_stride, dst_head_stride;
  int first;                              // index of its first head among all groups' heads
  int rotate;
  int cached;                             // dst is a cache: the token's page and slot give the place
};

struct Params {
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
  float sign;
  int32_t* status;
};

template <typename T, int N> struct alignas(sizeof(T) * N) Vec { T v[N]; };
template <int N> struct alignas(N * 4 > 16 ? 16 : N * 4) Floats { float v[N]; };

// What becomes of a token.
enum Fate { kDone = 0, kZeros = 1, kNaNs = 2 };

// Where token t stands: its position, and its page and slot where a cache is written.
template <bool APPEND>
__device__ __forceinline__ Fate place_of(const Params& p, int t, bool report, int* pos, int* page, int* slot) {
  *pos = *page = *slot = 0;
  Fate fate = kDone;
  if constexpr (APPEND) {
    int seq = t, behind = 1;              // tokens from this one to the end of its sequence, itself among them
    if (p.cu != nullptr) {
      seq = find_segment(p.cu, p.n_seg, t);
      behind = p.cu[seq + 1] - t;
    }
    if (behind < 1) return kZeros;        // behind the last sequence
    const int len = p.lens[seq];
    if (len == 0) return kZeros;          // a padding sequence
    *pos = len - behind;
    const int row = *pos / p.page_size;
    if (*pos < 0 || row >= p.max_pages || (p.cos != nullptr && *pos >= p.table_rows)) {
      fate = kNaNs;
    } else {
      *page = p.table[seq * p.table_stride + row];
      *slot = *pos - row * p.page_size;
      if (*page < 0 || *page >= p.num_pages) fate = kNaNs;
    }
  } else {
    if (p.positions != nullptr) {
      *pos = p.positions[t];
    } else {
      if (t >= p.cu[p.n_seg]) return kZeros;  // behind the last segment
      *pos = t - p.cu[find_segment(p.cu, p.n_seg, t)];
    }
    if (*pos < 0 || *pos >= p.table_rows) fate = kNaNs;
  }
  if (fate == kNaNs && report) report_error(p.status, kBadCacheIndex, APPEND ? kSiteAppend : kSiteRotary, t);
  return fate;
}

// Two vectors of VW elements rotated by VW angles: pair j is the two vectors' elements j, or (INTER) elements 2 j and 2 j + 1 of
// the two in a row.
template <typename T, int VW, bool INTER>
__device__ __forceinline__ void rotate(Vec<T, VW>& x, Vec<T, VW>& y, const float (&cs)[VW], const float (&sn)[VW]) {
  T in[2 * VW], to[2 * VW];
#pragma unroll
  for (int j = 0; j < VW; ++j) {
    in[j] = x.v[j];
    in[VW + j] = y.v[j];
  }
#pragma unroll
  for (int j = 0; j < VW; ++j) {
    const int i0 = INTER ? 2 * j : j, i1 = INTER ? 2 * j + 1 : VW + j;
    const float u = to_float(in[i0]), w = to_float(in[i1]);
    to[i0] = from_float<T>(u * cs[j] - w * sn[j]);
    to[i1] = from_float<T>(w * cs[j] + u * sn[j]);
  }
#pragma unroll
  for (int j = 0; j < VW; ++j) {
    x.v[j] = to[j];
    y.v[j] = to[VW + j];
  }
}

template <int VW>
__device__ __forceinline__ void load_angles(const float* c, const float* s, float sign, float (&cs)[VW], float (&sn)[VW]) {
  constexpr int N = VW > 4 ? 4 : VW;
#pragma unroll
  for (int j = 0; j < VW; j += N) {
    const Floats<N> a = *reinterpret_cast<const Floats<N>*>(c + j), b = *reinterpret_cast<const Floats<N>*>(s + j);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      cs[j + e] = a.v[e];
      sn[j + e] = sign * b.v[e];
    }
  }
}

// The kernel for long batches, whose token rows go through shared memory.  0 when it took the call, 1 when the call is not of its
// kind, negative for an error.
int launch_rows(Params& p, int vw, int dtype, bool inter, bool append, cudaStream_t s);

}  // namespace rotary
}  // namespace vafa
