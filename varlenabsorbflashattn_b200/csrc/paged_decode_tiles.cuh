// The tiles of paged decode attention: what a warp does with its keys of a block.
//
// All three keep, for each row of their row group, the running maximum m and sum l of the warp's own keys (log2 domain, fp32) and
// O = sum p v, rescaled when the maximum moves.  They differ in the products:
//   NarrowTile  16-bit, up to 8 rows: m16n8k16 with the keys (then the head dim) as the 16 rows of the product and the query rows as
//               its 8 columns.  One token of up to 8 grouped heads fills it, where a 128-row tcgen05 tile would be 1/128 to
//               1/16 full; a K or V element meets 8 rows, far below any tensor limit, so that HBM bounds it.
//   WideTile    16-bit, more rows (several tokens, many grouped heads): the query rows as the 16 rows of the product, so that P goes
//               from one product to the next in registers and statistics are kept for 2 rows a thread instead of 4.
//   Fp32Tile    fp32 multiply-adds (tensor products of fp32 would round to tf32), 4 or 8 rows: 4 lanes a key for the scores, then
//               the head dim over the lanes for P V.
// 16-bit P is split into two pieces (hi + lo) for the second product: one piece would put an error of the size of the output's own
// rounding on top of it (2.4e-3 instead of 1.7e-3 of bf16 outputs); the second costs a product per V fragment and no time that shows.
// fp16 P is held larger than it is, for its short range (kLift).
// Keys that some rows see and others do not (the new tokens themselves) are summed apart where V is not finite: 0 times a
// NaN would reach the rows that do not see it.  An infinite V that a row sees may come out of the two pieces of P as inf - inf or 0 inf;
// such a sum is NaN, and once the warps are joined its infinite addends decide it (bad_values in paged_decode.cuh).
#pragma once
#include <type_traits>

#include "paged_kernels.cuh"

namespace vafa {
namespace paged {

struct DecodeParams {
  const void* q; const void* k; const void* v;
  void* o; float* lse;
  const int32_t* lens; const int32_t* table;
  int64_t q_seq, q_token, q_head;
  int64_t k_page, k_slot, k_head, v_page, v_slot, v_head;
  int64_t table_stride;
  int n_seq, T, H, H_kv, g, R;            // g = H / H_kv, R = T * g rows of a unit
  int row_tiles, num_pages, page_size;
  uint32_t page_mul; int page_shift;      // j / page_size = (j * page_mul) >> 32 >> page_shift for j below 2^31 (page_mul 0: a shift alone)
  int capacity;                           // keys that a row of the page table holds
  float scale_log2;
  float* part_o; float2* part_ml; int4* meta;
  int32_t* status;
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// 16 bytes to shared memory; zeros where there is nothing to read.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool real) {
  const int n = real ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n));  // (no memory clobber: the places of later rows may be read meanwhile)
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm2(uint32_t& r0, uint32_t& r1, uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];" : "=r"(r0), "=r"(r1) : "r"(a) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (sizeof(T) == 2) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
      asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                   : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
      asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                   : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}
// Whether one of two 16-bit values is infinite or NaN: its exponent is all ones.
template <typename T>
__device__ __forceinline__ bool not_finite2(uint32_t x) {
  constexpr uint32_t e = sizeof(T) == 2 && std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  return (x & e) == e || (x & (e << 16)) == (e << 16);
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The weight of a partial sum with maximum m beside a maximum `all`: nothing where there is nothing.
__device__ __forceinline__ float weight(float m, float all) { return m == -INFINITY ? 0.f : exp2_approx(m - all); }

template <typename T>
__device__ __forceinline__ void store4(T* dst, float4 x) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(dst) = x;
  else *reinterpret_cast<uint2*>(dst) = make_uint2(pack2_out<T>(x.x, x.y), pack2_out<T>(x.z, x.w));
}
// Four values of a finished row.  A row that sees no key is zero; one whose every score is -inf is 0 / 0, as in the formula.
template <typename T>
__device__ __forceinline__ void write_row(const DecodeParams& p, int seq, int h, int r, int len, int D, int d, float4 sum, float m, float l) {
  const int t = r / p.g;
  const int64_t row = ((int64_t)seq * p.T + t) * p.H + h * p.g + r - t * p.g;
  const bool sees = len - p.T + t + 1 > 0;
  const float inv = 1.f / l;
  store4(reinterpret_cast<T*>(p.o) + row * D + d,
         sees ? make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv) : make_float4(0.f, 0.f, 0.f, 0.f));
  if (p.lse != nullptr && d == 0) p.lse[row] = sees ? (m + log2f(l)) * 0.69314718055994531f : -INFINITY;
}

// A block of keys as a tile sees it.
struct BlockView {
  unsigned char* k;        // the block's keys and values in shared memory
  unsigned char* v;
  int first;               // number of the block's first key in its sequence
  int len;                 // keys of the sequence
  int every;               // keys below this one are seen by every row
  bool masked;             // some key of the block is not seen by some row
};

// What a warp is: keys key0 .. key0 + KPW of a block, rows rg * ROWS_G .. of the tile.
struct Place { int lane, kw, rg; };

// Keys that a row (of the unit) sees.
__device__ __forceinline__ int row_limit(const DecodeParams& p, int len, int r) { return min(len, len - p.T + min(r, p.R - 1) / p.g + 1); }

template <typename T>
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack2_out<T>(a, b);
  const T* const h = reinterpret_cast<const T*>(&hi);
  lo = pack2_out<T>(a - to_float(h[0]), b - to_float(h[1]));
}

// fp16 has no value below 2^-24, and none with all its bits below 2^-14: weights far below the running maximum would lose bits, or
// be lost, in the second product although l has counted them (a first key 17 nats above 131 000 others that hold all of the
// values: 0.0078 for 0.0054; 17.4 nats: 0).  So P, and O with it, are held 2^15 times as large there, which no weight overflows; and where
// a row's largest weight among the warp's keys of a block is below 2^-8, they are lifted by that as well, O brought to the same scale
// for the block's products and back.  Powers of two: nothing is rounded.  O stays below 2^122: 2^31 keys, values of 2^16, 2^15, 2^60.
// What a weight can lose is then 2^-40 of the largest one that the warp has at once, with the keys beside it.
// (Without | with, us: 64 caches of 1k to 16k keys, 32 query and 8 K/V heads of 128 370 | 370, also where every block is lifted;
// 64 of 4k to 8k, four tokens of 4 grouped heads 256.5 | 257.9, of 8 333 | 336, seven of 8 527 | 536.)
template <typename T> constexpr int kLift = std::is_same<T, __half>::value ? 15 : 0;
__device__ __forceinline__ float pow2(int k) { return __int_as_float((127 + k) << 23); }
// `top`: the largest score of the keys, `now`: the running maximum.  (Not where there is no score, nor where every weight is zero.)
__device__ __forceinline__ int lift_of(float top, float now) {
  const float gap = now - top;
  return gap > 8.f && gap < 150.f ? (int)fminf(gap, 60.f) : 0;
}

template <typename C>
struct NarrowTile {
  using T = typename C::T;
  static constexpr int D = C::D, KT = C::KPW / 16;
  static constexpr int kAhead = D / 16 < 8 / KT ? D / 16 : 8 / KT;  // steps of the head dim on their way, for K and for V
  float o[D / 16][4];         // head dim 16 d + lane / 4 (+ 8), rows 2 (lane % 4) + {0, 1}
  float m[2], l[2];
  int limit[2];
  uint32_t qf[D / 16][2];
  int lane, key0, k_row, k_key, v_row, v_key, rg;

  __device__ __forceinline__ explicit NarrowTile(const Place& w) : lane(w.lane), key0(w.kw * C::KPW), rg(w.rg) {
    k_row = (key0 + (lane & 15)) * C::PITCH;
    k_key = C::key(lane & 15);
    v_row = (key0 + (lane & 7) + ((lane >> 4) & 1) * 8) * C::PITCH;
    v_key = C::key((lane & 7) + ((lane >> 4) & 1) * 8);
  }

  __device__ __forceinline__ void begin(const DecodeParams& p, const unsigned char* q, int len, int row0, float*) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      m[x] = -INFINITY;
      l[x] = 0.f;
      limit[x] = row_limit(p, len, row0 + rg * 8 + 2 * (lane & 3) + x);
    }
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
#pragma unroll
      for (int x = 0; x < 4; ++x) o[d][x] = 0.f;
      ldsm2(qf[d][0], qf[d][1], smem_addr(q) + (rg * 8 + (lane & 7)) * C::PITCH + (((2 * d + ((lane >> 3) & 1)) ^ C::key(lane & 7)) << 4));
    }
  }

  __device__ __forceinline__ void block(const DecodeParams& p, const BlockView& b) {
    const uint32_t ks = smem_addr(b.k) + k_row, vs = smem_addr(b.v) + v_row;
    // K fragments are on their way before the first product, V's first ones before the softmax; with one tile of keys even and odd
    // steps of the head dim are summed apart, which halves the chain of dependent products
    float s[KT][4], odd[4] = {0.f, 0.f, 0.f, 0.f};  // key 16 t + lane / 4 (+ 8 for x >= 2), rows 2 (lane % 4) + {0, 1}
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int x = 0; x < 4; ++x) s[t][x] = 0.f;
#pragma unroll
    for (int d0 = 0; d0 < D / 16; d0 += kAhead) {
      uint32_t a[KT][kAhead][4];
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int d = 0; d < kAhead; ++d) ldsm4(a[t][d], ks + t * 16 * C::PITCH + (((2 * (d0 + d) + (lane >> 4)) ^ k_key) << 4));
#pragma unroll
      for (int d = 0; d < kAhead; ++d)
#pragma unroll
        for (int t = 0; t < KT; ++t) mma<T>(KT == 1 && (d & 1) ? odd : s[t], a[t][d], qf[d0 + d][0], qf[d0 + d][1]);
    }
    uint32_t va[kAhead][4];
#pragma unroll
    for (int d = 0; d < kAhead; ++d) ldsm4t(va[d], vs + (((2 * d + ((lane >> 3) & 1)) ^ v_key) << 4));

    const int j0 = b.first + key0 + (lane >> 2);
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        s[t][x] = (KT == 1 ? s[t][x] + odd[x] : s[t][x]) * p.scale_log2;
        if (b.masked && (j0 + 16 * t + (x >> 1) * 8 >= limit[x & 1])) s[t][x] = -INFINITY;
      }
    float alpha[2];
    int lift[2];
    bool moved = false, far = false;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float top = fmaxf(s[0][x], s[0][x + 2]);
#pragma unroll
      for (int t = 1; t < KT; ++t) top = fmaxf(top, fmaxf(s[t][x], s[t][x + 2]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
      const float now = fmaxf(m[x], top);
      moved |= now != m[x];
      alpha[x] = weight(m[x], now);
      const float ref = now == -INFINITY ? 0.f : now;
      float sum = 0.f;
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        s[t][x] = exp2_approx(s[t][x] - ref);
        s[t][x + 2] = exp2_approx(s[t][x + 2] - ref);
        sum += s[t][x] + s[t][x + 2];
      }
      l[x] = l[x] * alpha[x] + sum;
      m[x] = now;
      if constexpr (kLift<T> != 0) {
        lift[x] = lift_of(top, now);
        far |= lift[x] != 0;
        alpha[x] *= pow2(lift[x]);
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          s[t][x] *= pow2(kLift<T> + lift[x]);
          s[t][x + 2] *= pow2(kLift<T> + lift[x]);
        }
      }
    }
    if (__any_sync(0xffffffffu, moved || far)) {
#pragma unroll
      for (int d = 0; d < D / 16; ++d)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[d][x] *= alpha[x & 1];
    }
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      // P as the second product's B operand: keys along k, rows along n
      uint32_t ph[2], pl[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        split2<T>(s[t][2 * e], s[t][2 * e + 1], ph[e], pl[e]);
        ph[e] = transpose8(ph[e]);
        pl[e] = transpose8(pl[e]);
      }
      const int first = b.first + key0 + 16 * t;
      const int apart0 = p.T > 1 && b.masked ? max(0, b.every - first) : 16;
      const int apart1 = min(16, b.len - first);
#pragma unroll
      for (int d0 = 0; d0 < D / 16; d0 += kAhead) {
        if (t > 0 || d0 > 0) {
#pragma unroll
          for (int d = 0; d < kAhead; ++d) ldsm4t(va[d], vs + t * 16 * C::PITCH + (((2 * (d0 + d) + ((lane >> 3) & 1)) ^ v_key) << 4));
        }
        bool apart = false;
        if (apart0 < apart1) {
#pragma unroll
          for (int d = 0; d < kAhead; ++d)
#pragma unroll
            for (int x = 0; x < 4; ++x) apart |= not_finite2<T>(va[d][x]);
          apart = __any_sync(0xffffffffu, apart);
        }
        if (apart) {  // V without those keys: a register holds the lane's pair of keys, or the pair 8 on
          const int a0 = 2 * (lane & 3);
          const uint32_t keep0 = (a0 < apart0 ? 0xffffu : 0u) | (a0 + 1 < apart0 ? 0xffff0000u : 0u);
          const uint32_t keep1 = (a0 + 8 < apart0 ? 0xffffu : 0u) | (a0 + 9 < apart0 ? 0xffff0000u : 0u);
#pragma unroll
          for (int d = 0; d < kAhead; ++d) {
            va[d][0] &= keep0;
            va[d][1] &= keep0;
            va[d][2] &= keep1;
            va[d][3] &= keep1;
          }
        }
#pragma unroll
        for (int d = 0; d < kAhead; ++d) mma<T>(o[d0 + d], va[d], ph[0], ph[1]);
#pragma unroll
        for (int d = 0; d < kAhead; ++d) mma<T>(o[d0 + d], va[d], pl[0], pl[1]);
        if (apart) {
          for (int k = apart0; k < apart1; ++k) {
            const unsigned char* const row = b.v + (key0 + 16 * t + k) * C::PITCH;
            const int ck = C::key(key0 + 16 * t + k);
            auto v_at = [&](int ch) { return to_float(reinterpret_cast<const T*>(row + (ch ^ ck) * 16)[lane >> 2]); };  // head dim 8 ch + lane / 4
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float w = __shfl_sync(0xffffffffu, k < 8 ? s[t][x] : s[t][x + 2], (k & 7) * 4 + (lane & 3));
              if (first + k < limit[x]) {
#pragma unroll
                for (int d = d0; d < d0 + kAhead; ++d) {
                  o[d][x] = fmaf(w, v_at(2 * d), o[d][x]);
                  o[d][x + 2] = fmaf(w, v_at(2 * d + 1), o[d][x + 2]);
                }
              }
            }
          }
        }
      }
    }
    if constexpr (kLift<T> != 0) {
      if (__any_sync(0xffffffffu, far)) {
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[d][x] *= pow2(-lift[x & 1]);
      }
    }
  }

  // the warp's (m, l) of its row group's rows
  __device__ __forceinline__ void stats(float2* out) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 4);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 8);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 16);
      if (lane < 4) out[2 * lane + x] = make_float2(m[x], l[x]);
    }
  }
  // eight rows of O
  __device__ __forceinline__ void rows(float* out, int) const {
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
#pragma unroll
      for (int x = 0; x < 4; ++x) out[(2 * (lane & 3) + (x & 1)) * C::MP + d * 16 + (lane >> 2) + (x >> 1) * 8] = o[d][x] * pow2(-kLift<T>);
  }
};

template <typename C>
struct WideTile {
  using T = typename C::T;
  static constexpr int D = C::D, KT = C::KPW / 16, NJ = 2 * KT;
  static constexpr int kMost = C::kRegisters < 200 || D == 256 ? 4 : 8;
  static constexpr int kAheadK = D / 16 < kMost / KT ? D / 16 : kMost / KT;  // steps of the head dim on their way, for K and for V
  static constexpr int kAheadV = D / 16 < kMost ? D / 16 : kMost;
  float o[D / 8][4];          // rows lane / 4 (+ 8 for x >= 2), head dim 8 n + 2 (lane % 4) + {0, 1}
  float m[2], l[2];
  int limit[2];
  uint32_t qf[C::kQReg ? D / 16 : 1][4];
  uint32_t q_at;
  int lane, key0, k_row, k_key, v_row, v_key, rg;

  __device__ __forceinline__ explicit WideTile(const Place& w) : lane(w.lane), key0(w.kw * C::KPW), rg(w.rg) {
    k_row = (key0 + (lane & 7) + ((lane >> 4) & 1) * 8) * C::PITCH;  // (keys 16 apart have the same key())
    k_key = C::key((lane & 7) + ((lane >> 4) & 1) * 8);
    v_row = (key0 + (lane & 15)) * C::PITCH;
    v_key = C::key(lane & 15);
  }
  __device__ __forceinline__ void q_frag(uint32_t (&a)[4], int d) const { ldsm4(a, q_at + (((2 * d + (lane >> 4)) ^ v_key) << 4)); }

  __device__ __forceinline__ void begin(const DecodeParams& p, const unsigned char* q, int len, int row0, float*) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      m[x] = -INFINITY;
      l[x] = 0.f;
      limit[x] = row_limit(p, len, row0 + rg * 16 + (lane >> 2) + 8 * x);
    }
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) o[n][x] = 0.f;
    q_at = smem_addr(q) + (rg * 16 + (lane & 15)) * C::PITCH;
    if constexpr (C::kQReg) {
#pragma unroll
      for (int d = 0; d < D / 16; ++d) q_frag(qf[d], d);
    }
  }

  __device__ __forceinline__ void block(const DecodeParams& p, const BlockView& b) {
    const uint32_t ks = smem_addr(b.k) + k_row, vs = smem_addr(b.v) + v_row;
    // s[j]: rows lane / 4 (+ 8 for x >= 2), keys 8 j + 2 (lane % 4) + {0, 1} of the warp's; with few keys even and odd steps of the
    // head dim are summed apart
    float s[NJ][4], odd[KT == 1 ? NJ : 1][4];
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        s[j][x] = 0.f;
        if (KT == 1) odd[j][x] = 0.f;
      }
#pragma unroll
    for (int d0 = 0; d0 < D / 16; d0 += kAheadK) {
      uint32_t kf[kAheadK][KT][4];
#pragma unroll
      for (int d = 0; d < kAheadK; ++d)
#pragma unroll
        for (int t = 0; t < KT; ++t)
          ldsm4(kf[d][t], ks + t * 16 * C::PITCH + (((2 * (d0 + d) + ((lane >> 3) & 1)) ^ k_key) << 4));
#pragma unroll
      for (int d = 0; d < kAheadK; ++d) {
        uint32_t a[4];
        if constexpr (!C::kQReg) q_frag(a, d0 + d);
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float(&to)[4] = KT == 1 && (d & 1) ? odd[KT == 1 ? e : 0] : s[2 * t + e];
            if constexpr (C::kQReg) mma<T>(to, qf[d0 + d], kf[d][t][2 * e], kf[d][t][2 * e + 1]);
            else mma<T>(to, a, kf[d][t][2 * e], kf[d][t][2 * e + 1]);
          }
      }
    }
    uint32_t va[kAheadV][4];
#pragma unroll
    for (int d = 0; d < kAheadV; ++d) ldsm4t(va[d], vs + (((2 * d + (lane >> 4)) ^ v_key) << 4));

    const int j0 = b.first + key0 + 2 * (lane & 3);
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        s[j][x] = (KT == 1 ? s[j][x] + odd[KT == 1 ? j : 0][x] : s[j][x]) * p.scale_log2;
        if (b.masked && (j0 + 8 * j + (x & 1) >= limit[x >> 1])) s[j][x] = -INFINITY;
      }
    float alpha[2];
    int lift[2];
    bool moved = false, far = false;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float top = fmaxf(s[0][2 * x], s[0][2 * x + 1]);
#pragma unroll
      for (int j = 1; j < NJ; ++j) top = fmaxf(top, fmaxf(s[j][2 * x], s[j][2 * x + 1]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float now = fmaxf(m[x], top);
      moved |= now != m[x];
      alpha[x] = weight(m[x], now);
      const float ref = now == -INFINITY ? 0.f : now;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[j][2 * x + e] = exp2_approx(s[j][2 * x + e] - ref);
          sum += s[j][2 * x + e];
        }
      l[x] = l[x] * alpha[x] + sum;
      m[x] = now;
      if constexpr (kLift<T> != 0) {
        lift[x] = lift_of(top, now);
        far |= lift[x] != 0;
        alpha[x] *= pow2(lift[x]);
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) s[j][2 * x + e] *= pow2(kLift<T> + lift[x]);
      }
    }
    if (__any_sync(0xffffffffu, moved || far)) {
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[n][x] *= alpha[x >> 1];
    }
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      uint32_t ph[4], pl[4];  // P as the second product's A operand
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int x = 0; x < 2; ++x) split2<T>(s[2 * t + e][2 * x], s[2 * t + e][2 * x + 1], ph[2 * e + x], pl[2 * e + x]);
      const int first = b.first + key0 + 16 * t;
      const int apart0 = p.T > 1 && b.masked ? max(0, b.every - first) : 16;
      const int apart1 = min(16, b.len - first);
#pragma unroll
      for (int d0 = 0; d0 < D / 16; d0 += kAheadV) {
        if (t > 0 || d0 > 0) {
#pragma unroll
          for (int d = 0; d < kAheadV; ++d) ldsm4t(va[d], vs + t * 16 * C::PITCH + (((2 * (d0 + d) + (lane >> 4)) ^ v_key) << 4));
        }
        bool apart = false;
        if (apart0 < apart1) {
#pragma unroll
          for (int d = 0; d < kAheadV; ++d)
#pragma unroll
            for (int x = 0; x < 4; ++x) apart |= not_finite2<T>(va[d][x]);
          apart = __any_sync(0xffffffffu, apart);
        }
        if (apart) {  // V without those keys: a register holds the lane's pair of keys, or the pair 8 on
          const int a0 = 2 * (lane & 3);
          const uint32_t keep0 = (a0 < apart0 ? 0xffffu : 0u) | (a0 + 1 < apart0 ? 0xffff0000u : 0u);
          const uint32_t keep1 = (a0 + 8 < apart0 ? 0xffffu : 0u) | (a0 + 9 < apart0 ? 0xffff0000u : 0u);
#pragma unroll
          for (int d = 0; d < kAheadV; ++d) {
            va[d][0] &= keep0;
            va[d][1] &= keep1;
            va[d][2] &= keep0;
            va[d][3] &= keep1;
          }
        }
#pragma unroll
        for (int d = 0; d < kAheadV; ++d)
#pragma unroll
          for (int e = 0; e < 2; ++e) mma<T>(o[2 * (d0 + d) + e], ph, va[d][2 * e], va[d][2 * e + 1]);
#pragma unroll
        for (int d = 0; d < kAheadV; ++d)
#pragma unroll
          for (int e = 0; e < 2; ++e) mma<T>(o[2 * (d0 + d) + e], pl, va[d][2 * e], va[d][2 * e + 1]);
        if (apart) {
          for (int k = apart0; k < apart1; ++k) {
            const unsigned char* const row = b.v + (key0 + 16 * t + k) * C::PITCH;
            const int ck = C::key(key0 + 16 * t + k);
            const int src = (lane & 28) | ((k & 7) >> 1);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float w0 = __shfl_sync(0xffffffffu, k < 8 ? s[2 * t][2 * x] : s[2 * t + 1][2 * x], src);
              const float w1 = __shfl_sync(0xffffffffu, k < 8 ? s[2 * t][2 * x + 1] : s[2 * t + 1][2 * x + 1], src);
              const float w = (k & 1) ? w1 : w0;
              if (first + k < limit[x]) {
#pragma unroll
                for (int n = 2 * d0; n < 2 * (d0 + kAheadV); ++n) {
                  const T* const v = reinterpret_cast<const T*>(row + (n ^ ck) * 16) + 2 * (lane & 3);
                  o[n][2 * x] = fmaf(w, to_float(v[0]), o[n][2 * x]);
                  o[n][2 * x + 1] = fmaf(w, to_float(v[1]), o[n][2 * x + 1]);
                }
              }
            }
          }
        }
      }
    }
    if constexpr (kLift<T> != 0) {
      if (__any_sync(0xffffffffu, far)) {
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[n][x] *= pow2(-lift[x >> 1]);
      }
    }
  }

  __device__ __forceinline__ void stats(float2* out) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
      if ((lane & 3) == 0) out[(lane >> 2) + 8 * x] = make_float2(m[x], l[x]);
    }
  }
  __device__ __forceinline__ void rows(float* out, int half) const {
#pragma unroll
    for (int n = 0; n < D / 8; ++n) {
      const float a = half ? o[n][2] : o[n][0], b = half ? o[n][3] : o[n][1];
      *reinterpret_cast<float2*>(out + (lane >> 2) * C::MP + 8 * n + 2 * (lane & 3)) = make_float2(a * pow2(-kLift<T>), b * pow2(-kLift<T>));
    }
  }
};

template <typename C>
struct Fp32Tile {
  static constexpr int D = C::D, KPW = C::KPW, KL = KPW / 8, DV = (D + 31) / 32;
  static constexpr int NR = C::ROWS_G, RL = NR / 4;  // rows of the warp, and of a lane where statistics are kept
  float o[NR][DV];            // rows 0 .. NR, head dim 128 (y / 4) + 4 lane + y % 4, or DV lane + y below 128
  float m[RL], l[RL];         // rows RL (lane % 4) .. + RL
  int limit[RL];
  const unsigned char* q_at;
  float* pr;                  // the warp's P [KPW][NR], then alpha and the limits of the rows
  int lane, key0, rg;

  __device__ __forceinline__ explicit Fp32Tile(const Place& w) : lane(w.lane), key0(w.kw * KPW), rg(w.rg) {}

  __device__ __forceinline__ void begin(const DecodeParams& p, const unsigned char* q, int len, int row0, float* scratch) {
    q_at = q + rg * NR * C::PITCH;
    pr = scratch;
#pragma unroll
    for (int x = 0; x < RL; ++x) {
      m[x] = -INFINITY;
      l[x] = 0.f;
      limit[x] = row_limit(p, len, row0 + rg * NR + RL * (lane & 3) + x);
    }
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int y = 0; y < DV; ++y) o[r][y] = 0.f;
  }

  __device__ __forceinline__ void block(const DecodeParams& p, const BlockView& b) {
    float s[KL][RL];  // key 8 e + lane / 4, the lane's rows
    {
      float acc[KL][NR];
#pragma unroll
      for (int e = 0; e < KL; ++e)
#pragma unroll
        for (int r = 0; r < NR; ++r) acc[e][r] = 0.f;
      const unsigned char* const kr = b.k + (key0 + (lane >> 2)) * C::PITCH;  // (keys 8 apart have the same key())
      const int ck = C::key(lane >> 2);
#pragma unroll 4
      for (int d = 0; d < D / 16; ++d) {
        float4 kv[KL];
#pragma unroll
        for (int e = 0; e < KL; ++e) kv[e] = *reinterpret_cast<const float4*>(kr + e * 8 * C::PITCH + ((4 * d + (lane & 3)) ^ ck) * 16);
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          const float4 qv = *reinterpret_cast<const float4*>(q_at + r * C::PITCH + ((4 * d + (lane & 3)) ^ C::key(r)) * 16);
#pragma unroll
          for (int e = 0; e < KL; ++e)
            acc[e][r] = fmaf(qv.x, kv[e].x, fmaf(qv.y, kv[e].y, fmaf(qv.z, kv[e].z, fmaf(qv.w, kv[e].w, acc[e][r]))));
        }
      }
      // the four lanes of a key sum their quarters and share out the rows
      const bool hi2 = (lane & 2) != 0, hi1 = (lane & 1) != 0;
#pragma unroll
      for (int e = 0; e < KL; ++e) {
        float half[NR / 2];
#pragma unroll
        for (int r = 0; r < NR / 2; ++r) {
          const float give = hi2 ? acc[e][r] : acc[e][r + NR / 2], keep = hi2 ? acc[e][r + NR / 2] : acc[e][r];
          half[r] = keep + __shfl_xor_sync(0xffffffffu, give, 2);
        }
#pragma unroll
        for (int r = 0; r < RL; ++r) {
          const float give = hi1 ? half[r] : half[r + RL], keep = hi1 ? half[r + RL] : half[r];
          s[e][r] = keep + __shfl_xor_sync(0xffffffffu, give, 1);
        }
      }
    }
    const int j0 = b.first + key0 + (lane >> 2);
    float alpha[RL];
    bool moved = false;
#pragma unroll
    for (int x = 0; x < RL; ++x) {
      float top = -INFINITY;
#pragma unroll
      for (int e = 0; e < KL; ++e) {
        s[e][x] *= p.scale_log2;
        if (b.masked && (j0 + 8 * e >= limit[x])) s[e][x] = -INFINITY;
        top = fmaxf(top, s[e][x]);
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
      const float now = fmaxf(m[x], top);
      moved |= now != m[x];
      alpha[x] = weight(m[x], now);
      const float ref = now == -INFINITY ? 0.f : now;
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < KL; ++e) {
        s[e][x] = exp2_approx(s[e][x] - ref);
        sum += s[e][x];
      }
      l[x] = l[x] * alpha[x] + sum;
      m[x] = now;
    }
    const int apart0 = p.T > 1 && b.masked ? max(0, b.every - (b.first + key0)) : KPW;
    __syncwarp();
#pragma unroll
    for (int x = 0; x < RL; ++x) {
#pragma unroll
      for (int e = 0; e < KL; ++e) pr[(8 * e + (lane >> 2)) * NR + RL * (lane & 3) + x] = s[e][x];
      if (lane < 4) {
        pr[KPW * NR + RL * lane + x] = alpha[x];
        reinterpret_cast<int*>(pr)[(KPW + 1) * NR + RL * lane + x] = limit[x];
      }
    }
    __syncwarp();
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const float f = pr[KPW * NR + r];
#pragma unroll
        for (int y = 0; y < DV; ++y) o[r][y] *= f;
      }
    }
    constexpr int W = D >= 128 ? 4 : D / 32 > 0 ? D / 32 : 1;  // floats of one read
    const unsigned char* const vr = b.v + key0 * C::PITCH;
    const bool has = D >= 32 || lane < D;
#pragma unroll 4
    for (int k = 0; k < KPW; ++k) {
      float pk[NR];
#pragma unroll
      for (int r = 0; r < NR; r += 4) {
        const float4 x = *reinterpret_cast<const float4*>(pr + k * NR + r);
        pk[r] = x.x; pk[r + 1] = x.y; pk[r + 2] = x.z; pk[r + 3] = x.w;
      }
      float v[DV];
      const unsigned char* const row = vr + k * C::PITCH;
      const int ck = C::key(k);
#pragma unroll
      for (int y = 0; y < DV; y += W) {
        const int ch = y * 8 + lane * W / 4;
        const float* const x = reinterpret_cast<const float*>(row + (ch ^ ck) * 16) + lane * W % 4;
        if constexpr (W == 4) {
          const float4 f = *reinterpret_cast<const float4*>(x);
          v[y] = f.x; v[y + 1] = f.y; v[y + 2] = f.z; v[y + 3] = f.w;
        } else if constexpr (W == 2) {
          const float2 f = *reinterpret_cast<const float2*>(x);
          v[y] = f.x; v[y + 1] = f.y;
        } else {
          v[y] = has ? *x : 0.f;
        }
      }
      if (k < apart0) {
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int y = 0; y < DV; ++y) o[r][y] = fmaf(pk[r], v[y], o[r][y]);
      } else {
        const int j = b.first + key0 + k;
#pragma unroll
        for (int r = 0; r < NR; ++r)
          if (j < reinterpret_cast<const int*>(pr)[(KPW + 1) * NR + r]) {
#pragma unroll
            for (int y = 0; y < DV; ++y) o[r][y] = fmaf(pk[r], v[y], o[r][y]);
          }
      }
    }
  }

  __device__ __forceinline__ void stats(float2* out) {
#pragma unroll
    for (int x = 0; x < RL; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 4);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 8);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 16);
      if (lane < 4) out[RL * lane + x] = make_float2(m[x], l[x]);
    }
  }
  __device__ __forceinline__ void rows(float* out, int) const {
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int y = 0; y < DV; ++y) {
        const int d = D >= 128 ? (y / 4) * 128 + lane * 4 + (y & 3) : lane * DV + y;
        if (d < D) out[r * C::MP + d] = o[r][y];
      }
  }
};

}  // namespace paged
}  // namespace vafa
