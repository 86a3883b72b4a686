// Attention of new tokens over a paged key/value cache.
//
// For a sequence and a K/V head, the rows r = t * g + j (token t, query head j of the g that share the K/V head) attend
// over the cache's keys:   o_r = sum_j p_rj v_j / sum_j p_rj,  p_rj = 2^(c q_r.k_j - m_r),  c = scale log2(e),
// with one pass over the keys, the running maximum m and the running sum kept in fp32.
//
// HBM bounds it: a K/V element is read once and meets a handful of rows.  So
//  - the keys of all (sequence, K/V head, row tile) units are one line of blocks of BK keys, cut into as many equal
//    pieces as there are CTAs, whatever the lengths are; a unit that lies in several pieces leaves partial results
//    (m, sum, sum p v) in the workspace and the combine kernel joins them in the order of the pieces, so the
//    result does not depend on timing.  Each CTA finds its piece from the lengths itself: nothing is read on the host.
//  - K and V blocks are copied to shared memory by cp.async, S blocks deep, 16 bytes at a time, because a page may
//    be of any size and end inside a block; page ids are read two blocks before they are needed.
//  - 16-bit types use m16n8k16 products with the keys (then the head dim) as their 16 rows and the query rows as their 8 columns:
//    a single token of up to 8 grouped heads fills the tile, where 128-row tcgen05 tiles would be 1/128 to 1/16 full.
//    The products are far from the tensor pipe's limit (see the table in the notes), so the legacy instruction costs nothing.
//  - each of the KW warps of a row group owns 16 (fp32: 8 or 16) keys of a block with its own maximum and sum, so the loop has no
//    exchange between warps; they are joined once, at the unit's end.
// P is split into two 16-bit pieces (hi + lo) for the second product: one piece would put an error of the size of the
// output's own rounding on top of it, the second costs one more product per V fragment and no time.
#pragma once
#include <atomic>
#include <type_traits>

#include "paged_kernels.cuh"
#include "profile.cuh"

#ifndef PD_CTAS
#define PD_CTAS 3
#endif
#ifndef PD_UNIT
#define PD_UNIT 2
#endif
#ifndef PD_KW
#define PD_KW 4
#endif
#ifndef PD_MAXS
#define PD_MAXS 6
#endif
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

template <typename T_, int D_, int NT_, int RG_, int KW_>
struct Config {
  using T = T_;
  static constexpr int D = D_, NT = NT_, RG = RG_, KW = KW_;
  static constexpr bool kFp32 = sizeof(T) == 4;
  static constexpr int KPW = kFp32 && D >= 128 ? 8 : 16;   // keys of a warp
  static constexpr int BK = KW * KPW;
  static constexpr int ROWS_G = 8 * NT, ROWS = ROWS_G * RG;
  static constexpr int THREADS = 32 * KW * RG;
  static constexpr int VEC = 16 / (int)sizeof(T), CH = D / VEC;
  // A row's 16-byte chunks are stored at chunk ^ key(row): the 8 rows that an ldmatrix tile (fp32: the 2 rows that 8 lanes)
  // read at the same chunk then lie in different banks without padding.
  static constexpr int PITCH = D * (int)sizeof(T);
  static __device__ __forceinline__ int key(int row) {
    if constexpr (kFp32) return CH >= 8 ? (row & 1) * 4 : 0;
    else return (row / (CH < 8 ? 8 / CH : 1)) & ((CH < 8 ? CH : 8) - 1);
  }
  static constexpr int kStageBytes = (2 * BK + ROWS) * PITCH;
  static constexpr bool kQReg = !kFp32 && (RG == 1 || (RG == 2 && D <= 64));  // Q fragments stay in registers
  static constexpr int kQBytes = kQReg ? 0 : ROWS * PITCH;
  static constexpr int MP = D + 4;                         // pitch of the join buffer, floats: 8 rows of each warp of a row group
  static constexpr int kJoinBytes = KW * 8 * MP * 4;
  static_assert(kJoinBytes <= kStageBytes, "the join buffer takes the place of a stage that has been read");
  static constexpr int kMlBytes = RG * KW * ROWS_G * 8;
  static constexpr int kPBytes = kFp32 ? RG * KW * (KPW + 2) * 8 * 4 : 0;
  static constexpr int kBudget = 227 * 1024;
  static constexpr int kMaxStages = PD_MAXS;
  static constexpr int bytes_of(int s) { return s * kStageBytes + kQBytes + kMlBytes + kPBytes + (s + 2) * (16 + BK * 16) + 256; }
  static constexpr int fit(int ctas) {
    int s = kMaxStages;
    while (s > 1 && (bytes_of(s) + 1024) * ctas > kBudget + 1024) --s;
    return s;
  }
  // CTAs of an SM, as far as registers and shared memory go
  static constexpr int CTAS = RG == 1 && NT == 1 && fit(PD_CTAS) >= 2 ? PD_CTAS : RG <= 2 && !(D == 256) && fit(2) >= 2 ? 2 : 1;
  static constexpr int S = fit(CTAS);
  static constexpr int kInfo = S + 2;                      // slots of the ring of block descriptions
  static_assert(S >= 2, "no room for two stages");
  static constexpr int kSmem = bytes_of(S);
};

// A piece of the line of blocks: what a CTA needs to know to find its first block.  A unit costs more than its blocks (its
// queries, the join of the warps, the rows' way out), so the line that is cut has `kUnitCost` slots more in front of each
// unit's blocks; a piece that begins or ends among those begins or ends with the unit's first block.
constexpr int kUnitCost = PD_UNIT;
struct Piece {
  long long first, last;      // blocks [first, last), the slots not counted
  long long share;            // slots and blocks of a piece
  int seq, unit, kb;          // the first one's sequence, its unit of the sequence's and its block of the unit's
};

__device__ __forceinline__ int clamped_len(const DecodeParams& p, int s) {
  const int len = p.lens[s];
  return len < 0 ? 0 : len > p.capacity ? p.capacity : len;
}
// A sequence without keys has a block too: its rows are written.
template <int BK>
__device__ __forceinline__ int blocks_of(int len) { return len <= 0 ? 1 : (len + BK - 1) / BK; }

// Cuts the line.  Every thread takes a run of sequences; a scan of the runs' sums, and the threads whose runs hold the two ends
// of the piece look for them.
template <typename C>
__device__ void find_piece(const DecodeParams& p, Piece* out, long long* scan, int min_share) {
  constexpr int kWarps = C::THREADS / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int each = (p.n_seq + C::THREADS - 1) / C::THREADS;
  const int s0 = min(p.n_seq, tid * each), s1 = min(p.n_seq, s0 + each);
  const int per_seq = p.H_kv * p.row_tiles;
  long long mine = 0;
  for (int s = s0; s < s1; ++s) {
    mine += blocks_of<C::BK>(clamped_len(p, s)) + kUnitCost;
    if (p.lens[s] < 0 || p.lens[s] > p.capacity) report_error(p.status, kBadCacheIndex, kSiteDecode, s);
  }
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  if (lane == 31) scan[warp] = incl;
  __syncthreads();
  long long before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += scan[w];
    total += scan[w];
  }
  incl += before;
  total *= per_seq;
  // (as many slots as 32 bits hold are cut with a short division)
  long long share = total < 0x7fffffff ? ((uint32_t)total + gridDim.x - 1) / gridDim.x : (total + gridDim.x - 1) / gridDim.x;
  if (share < min_share) share = min_share;
#pragma unroll
  for (int end = 0; end < 2; ++end) {
    const long long target = min(total, (blockIdx.x + end) * share);
    long long at = (incl - mine) * per_seq;
    if (target >= at && target < incl * per_seq) {
      int s = s0, len_u = 0;
      for (; s < s1; ++s) {
        len_u = blocks_of<C::BK>(clamped_len(p, s)) + kUnitCost;
        if (target < at + (long long)len_u * per_seq) break;
        at += (long long)len_u * per_seq;
      }
      const int rest = (int)(target - at), unit = rest / len_u, kb = max(0, rest - unit * len_u - kUnitCost);
      const long long block = at - (long long)kUnitCost * s * per_seq + (long long)unit * (len_u - kUnitCost) + kb;
      if (end == 0) {
        out->first = block;
        out->seq = s;
        out->unit = unit;
        out->kb = kb;
      } else {
        out->last = block;
      }
    } else if (target == total && tid == 0) {
      (end == 0 ? out->first : out->last) = total - (long long)kUnitCost * p.n_seq * per_seq;
    }
  }
  if (tid == 0) out->share = share;
  __syncthreads();
}

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

__device__ __forceinline__ int page_of(const DecodeParams& p, int j) {
  return p.page_mul ? (int)(__umulhi((uint32_t)j, p.page_mul) >> p.page_shift) : j >> p.page_shift;
}

struct Block {  // a block of the line, as its ring slot describes it
  int seq, hr, kb, len;   // hr: K/V head, and row tile in the upper half
};

template <typename C>
__global__ void __launch_bounds__(C::THREADS, C::CTAS) decode_kernel(const DecodeParams p, int min_share) {
  using T = typename C::T;
  constexpr int D = C::D, NT = C::NT, RG = C::RG, BK = C::BK, KW = C::KW, S = C::S, KPW = C::KPW;
  constexpr bool kFp32 = C::kFp32;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ Piece piece;
  __shared__ long long scan[C::THREADS / 32];

  unsigned char* const stages = smem;
  unsigned char* at = smem + S * C::kStageBytes;
  unsigned char* const q_now = at;                     at += C::kQBytes;
  float2* const join_ml = reinterpret_cast<float2*>(at); at += C::kMlBytes;
  float* const p_all = reinterpret_cast<float*>(at);   at += C::kPBytes;
  at = smem + (((at - smem) + 15) & ~15);
  longlong2* const row_at = reinterpret_cast<longlong2*>(at); at += C::kInfo * BK * 16;
  Block* const info = reinterpret_cast<Block*>(at);

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int kw = warp % KW, rg = warp / KW;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  find_piece<C>(p, &piece, scan, min_share);
  const long long first = piece.first;
  const int n_iter = (int)(piece.last - first);
  if (tid == 0) p.meta[blockIdx.x] = make_int4(-1, 0, 0, 0);
  if (n_iter <= 0) return;

  // ---- the walk along the line: the threads below BK look up the places of the keys of one block after the other ----
  int w_seq = piece.seq, w_len = clamped_len(p, w_seq), w_nb = blocks_of<BK>(w_len);
  int w_h = piece.unit / p.row_tiles, w_rt = piece.unit - w_h * p.row_tiles, w_kb = piece.kb;
  const bool looks_up = tid < BK;
  auto walk = [&]() {
    if (++w_kb == w_nb) {
      w_kb = 0;
      if (++w_rt == p.row_tiles) {
        w_rt = 0;
        if (++w_h == p.H_kv) {
          w_h = 0;
          if (++w_seq < p.n_seq) {
            w_len = clamped_len(p, w_seq);
            w_nb = blocks_of<BK>(w_len);
          }
        }
      }
    }
  };
  // a lookup under way: the page id is on its way into `page` until land() is called
  struct Lookup { Block b; int page, slot; };
  auto start = [&](Lookup& x) {
    x.b = Block{w_seq, w_h | (w_rt << 16), w_kb, w_len};
    x.page = -1;
    x.slot = 0;
    if (w_seq < p.n_seq) {
      const int j = w_kb * BK + tid;
      if (j < w_len) {
        const int row = page_of(p, j);
        x.slot = j - row * p.page_size;
        x.page = __ldg(p.table + w_seq * p.table_stride + row);
      }
    }
  };
  auto land = [&](const Lookup& x, int i) {
    const int slot = i % C::kInfo;
    if (tid == 0) info[slot] = x.b;
    longlong2 r = make_longlong2(-1, -1);
    if (x.b.seq < p.n_seq && x.b.kb * BK + tid < x.b.len) {
      if (x.page >= 0 && x.page < p.num_pages)
        r = make_longlong2(x.page * p.k_page + x.slot * p.k_slot, x.page * p.v_page + x.slot * p.v_slot);
      else
        report_error(p.status, kBadCacheIndex, kSiteDecode, x.b.seq);
    }
    row_at[slot * BK + tid] = r;
  };
  // copies block i (of this CTA) into its stage
  auto issue = [&](int i) {
    const Block b = info[i % C::kInfo];
    const longlong2* const rows = row_at + (i % C::kInfo) * BK;
    const int h = b.hr & 0xffff;
    unsigned char* const st = stages + (i % S) * C::kStageBytes;
    const T* const kh = reinterpret_cast<const T*>(p.k) + h * p.k_head;
    const T* const vh = reinterpret_cast<const T*>(p.v) + h * p.v_head;
    const uint32_t ks = smem_addr(st), vs = ks + BK * C::PITCH, qs = vs + BK * C::PITCH;
#pragma unroll
    for (int x = 0; x < (BK * C::CH + C::THREADS - 1) / C::THREADS; ++x) {
      const int e = x * C::THREADS + tid;
      if ((BK * C::CH) % C::THREADS != 0 && e >= BK * C::CH) break;
      const int row = e / C::CH, ch = e % C::CH;
      const longlong2 r = rows[row];
      const bool real = r.x >= 0;
      const int to = row * C::PITCH + (ch ^ C::key(row)) * 16;
      copy16(ks + to, kh + (real ? r.x + ch * C::VEC : 0), real);
      copy16(vs + to, vh + (real ? r.y + ch * C::VEC : 0), real);
    }
    if (i == 0 || b.kb == 0) {
      const int row0 = (b.hr >> 16) * C::ROWS;
      const T* const qb = reinterpret_cast<const T*>(p.q) + b.seq * p.q_seq;
      for (int e = tid; e < C::ROWS * C::CH; e += C::THREADS) {
        const int row = e / C::CH, ch = e % C::CH, r = row0 + row;
        const bool real = r < p.R;
        const int t = real ? r / p.g : 0;
        copy16(qs + row * C::PITCH + (ch ^ C::key(row)) * 16, qb + (real ? t * p.q_token + (h * p.g + r - t * p.g) * p.q_head + ch * C::VEC : 0), real);
      }
    }
  };

  if (looks_up) {
    Lookup x[S + 1];
#pragma unroll
    for (int i = 0; i < S; ++i) {
      start(x[i]);
      walk();
    }
#pragma unroll
    for (int i = 0; i < S; ++i) land(x[i], i);
  }
  Lookup next;
  if (looks_up) {
    start(next);  // of block S
    walk();
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < S - 1; ++i) {
    if (i < n_iter) issue(i);
    copy_commit();
  }

  // ---- state of the unit under way ----
  float o[kFp32 ? 8 : D / 16 * NT][kFp32 ? (D + 31) / 32 : 4];
  float m[2 * NT], l[2 * NT];          // of the columns (rows of the unit) 8 nt + 2 (lane % 4) + {0, 1}
  int limit[2 * NT];                   // keys that the row sees
  uint32_t qf[C::kQReg ? D / 16 : 1][NT][2];
  constexpr int kMost = C::THREADS * C::CTAS >= 512 ? 4 : 8;
  constexpr int kAhead = D / 16 < kMost ? D / 16 : kMost;      // fragments of K or V in flight, as registers allow
  const int key0 = kw * KPW;                                   // the warp's keys of a block
  const int k_row = (key0 + (lane & 15)) * C::PITCH, k_key = C::key(lane & 15);
  const int v_row = (key0 + (lane & 7) + ((lane >> 4) & 1) * 8) * C::PITCH, v_key = C::key((lane & 7) + ((lane >> 4) & 1) * 8);
  auto q_addr = [&](uint32_t base, int nt, int d) {
    return base + (rg * C::ROWS_G + nt * 8 + (lane & 7)) * C::PITCH + (((2 * d + ((lane >> 3) & 1)) ^ C::key(lane & 7)) << 4);
  };
  float* const p_warp = p_all + warp * (KPW + 2) * 8;
  int unit_kb0 = 0;                    // first block of the unit that this CTA has

  for (int i = 0; i < n_iter; ++i) {
    copy_wait<S - 2>();
    __syncthreads();
    if (i + S - 1 < n_iter) issue(i + S - 1);
    copy_commit();
    if (looks_up) {
      land(next, i + S);
      start(next);
      walk();
    }
    const Block b = info[i % C::kInfo];
    unsigned char* const st = stages + (i % S) * C::kStageBytes;
    const uint32_t ks = smem_addr(st), vs = ks + BK * C::PITCH, qs = vs + BK * C::PITCH;
    const int nb = blocks_of<BK>(b.len);
    const int h = b.hr & 0xffff, row0 = (b.hr >> 16) * C::ROWS;

    if (i == 0 || b.kb == 0) {
      unit_kb0 = b.kb;
#pragma unroll
      for (int x = 0; x < 2 * NT; ++x) {
        m[x] = -INFINITY;
        l[x] = 0.f;
        const int r = row0 + rg * C::ROWS_G + (x >> 1) * 8 + 2 * (lane & 3) + (x & 1);
        limit[x] = min(b.len, b.len - p.T + min(r, p.R - 1) / p.g + 1);
      }
#pragma unroll
      for (int x = 0; x < (int)(sizeof(o) / sizeof(o[0])); ++x)
#pragma unroll
        for (int y = 0; y < (int)(sizeof(o[0]) / 4); ++y) o[x][y] = 0.f;
      if constexpr (C::kQReg) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int d = 0; d < D / 16; ++d)
            ldsm2(qf[d][nt][0], qf[d][nt][1], q_addr(qs, nt, d));
      } else {
        for (int e = tid; e < C::ROWS * C::CH; e += C::THREADS) {
          *reinterpret_cast<uint4*>(q_now + e * 16) = *reinterpret_cast<const uint4*>(st + 2 * BK * C::PITCH + e * 16);
        }
        __syncthreads();
      }
    }

    // ---- scores: s[nt][2 e + x] = key 8 e + lane / 4 of the warp's, column 8 nt + 2 (lane % 4) + x ----
    float s[NT][4];
    if constexpr (kFp32) {
      constexpr int KL = KPW / 8;
      float acc[KL][8];
#pragma unroll
      for (int e = 0; e < KL; ++e)
#pragma unroll
        for (int r = 0; r < 8; ++r) acc[e][r] = 0.f;
      const unsigned char* const kr = st + (key0 + (lane >> 2)) * C::PITCH;  // (keys 8 apart have the same key())
      const unsigned char* const qr = q_now + rg * 8 * C::PITCH;
      const int ck = C::key(lane >> 2);
#pragma unroll 4
      for (int d = 0; d < D / 16; ++d) {
        float4 kv[KL];
#pragma unroll
        for (int e = 0; e < KL; ++e) kv[e] = *reinterpret_cast<const float4*>(kr + e * 8 * C::PITCH + ((4 * d + (lane & 3)) ^ ck) * 16);
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const float4 qv = *reinterpret_cast<const float4*>(qr + r * C::PITCH + ((4 * d + (lane & 3)) ^ C::key(r)) * 16);
#pragma unroll
          for (int e = 0; e < KL; ++e)
            acc[e][r] = fmaf(qv.x, kv[e].x, fmaf(qv.y, kv[e].y, fmaf(qv.z, kv[e].z, fmaf(qv.w, kv[e].w, acc[e][r]))));
        }
      }
      // the four lanes of a key sum their quarters; lane % 4 keeps rows 2 (lane % 4) and the next
#pragma unroll
      for (int e = 0; e < KL; ++e) {
        float h4[4];
        const bool hi2 = (lane & 2) != 0, hi1 = (lane & 1) != 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float give = hi2 ? acc[e][r] : acc[e][r + 4], keep = hi2 ? acc[e][r + 4] : acc[e][r];
          h4[r] = keep + __shfl_xor_sync(0xffffffffu, give, 2);
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float give = hi1 ? h4[r] : h4[r + 2], keep = hi1 ? h4[r + 2] : h4[r];
          s[0][2 * e + r] = keep + __shfl_xor_sync(0xffffffffu, give, 1);
        }
      }
      if constexpr (KL == 1) s[0][2] = s[0][3] = -INFINITY;
    } else {
      // K fragments are all on their way before the first product, V's first ones before the softmax; even and odd steps of the
      // head dim are summed apart, which halves the chain of dependent products
      float odd[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 4; ++x) s[nt][x] = odd[nt][x] = 0.f;
#pragma unroll
      for (int d0 = 0; d0 < D / 16; d0 += kAhead) {
        uint32_t a[kAhead][4];
#pragma unroll
        for (int d = 0; d < kAhead; ++d)
          ldsm4(a[d], ks + k_row + (((2 * (d0 + d) + (lane >> 4)) ^ k_key) << 4));
#pragma unroll
        for (int d = 0; d < kAhead; ++d)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            uint32_t b0, b1;
            if constexpr (C::kQReg) {
              b0 = qf[d0 + d][nt][0];
              b1 = qf[d0 + d][nt][1];
            } else {
              ldsm2(b0, b1, q_addr(smem_addr(q_now), nt, d0 + d));
            }
            mma<T>((d & 1) ? odd[nt] : s[nt], a[d], b0, b1);
          }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 4; ++x) s[nt][x] += odd[nt][x];
    }
    uint32_t va[kFp32 ? 1 : kAhead][4];
    if constexpr (!kFp32) {
#pragma unroll
      for (int d = 0; d < kAhead; ++d) ldsm4t(va[d], vs + v_row + (((2 * d + ((lane >> 3) & 1)) ^ v_key) << 4));
    }

    // ---- softmax ----
    const int j0 = b.kb * BK + key0 + (lane >> 2);                // the lane's first key
    const int every = b.len - p.T + 1;                            // keys below this one are seen by every row
    const bool masked = (b.kb + 1) * BK > every;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        s[nt][x] *= p.scale_log2;
        if (masked && (j0 + (x >> 1) * 8 >= limit[2 * nt + (x & 1)])) s[nt][x] = -INFINITY;
        if (kFp32 && KPW == 8 && x >= 2) s[nt][x] = -INFINITY;
      }
    float alpha[2 * NT];
    bool moved = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float top = fmaxf(s[nt][x], s[nt][x + 2]);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
        const int c = 2 * nt + x;
        const float now = fmaxf(m[c], top);
        moved |= now != m[c];
        alpha[c] = weight(m[c], now);
        const float ref = now == -INFINITY ? 0.f : now;
        s[nt][x] = exp2_approx(s[nt][x] - ref);
        s[nt][x + 2] = exp2_approx(s[nt][x + 2] - ref);
        l[c] = l[c] * alpha[c] + (s[nt][x] + s[nt][x + 2]);
        m[c] = now;
      }

    // ---- O = alpha O + P V ----
    // Keys that some rows see and others do not are summed apart where V is not finite: 0 times a NaN would reach the others.
    const int apart0 = p.T > 1 && masked ? max(0, every - (b.kb * BK + key0)) : KPW;
    const int apart1 = min(KPW, b.len - (b.kb * BK + key0));
    if constexpr (kFp32) {
      constexpr int DV = (D + 31) / 32;
      float* const pr = p_warp;
      __syncwarp();
#pragma unroll
      for (int e = 0; e < KPW / 8; ++e)
        *reinterpret_cast<float2*>(pr + (8 * e + (lane >> 2)) * 8 + 2 * (lane & 3)) = make_float2(s[0][2 * e], s[0][2 * e + 1]);
      if (lane < 4) *reinterpret_cast<float2*>(pr + KPW * 8 + 2 * lane) = make_float2(alpha[0], alpha[1]);
      if (lane < 4) *reinterpret_cast<int2*>(pr + (KPW + 1) * 8 + 2 * lane) = make_int2(limit[0], limit[1]);
      __syncwarp();
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const float f = pr[KPW * 8 + r];
#pragma unroll
          for (int y = 0; y < DV; ++y) o[r][y] *= f;
        }
      }
      constexpr int W = D >= 128 ? 4 : D / 32 > 0 ? D / 32 : 1;  // floats of one read
      const unsigned char* const vr = st + (BK + key0) * C::PITCH;
      const bool has = D >= 32 || lane < D;
#pragma unroll 4
      for (int k = 0; k < KPW; ++k) {
        const float4 pa = *reinterpret_cast<const float4*>(pr + k * 8), pb = *reinterpret_cast<const float4*>(pr + k * 8 + 4);
        const float pk[8] = {pa.x, pa.y, pa.z, pa.w, pb.x, pb.y, pb.z, pb.w};
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
          for (int r = 0; r < 8; ++r)
#pragma unroll
            for (int y = 0; y < DV; ++y) o[r][y] = fmaf(pk[r], v[y], o[r][y]);
        } else {
          const int j = b.kb * BK + key0 + k;
#pragma unroll
          for (int r = 0; r < 8; ++r)
            if (j < reinterpret_cast<const int*>(pr)[(KPW + 1) * 8 + r]) {
#pragma unroll
              for (int y = 0; y < DV; ++y) o[r][y] = fmaf(pk[r], v[y], o[r][y]);
            }
        }
      }
    } else {
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[d * NT + nt][x] *= alpha[2 * nt + (x & 1)];
      }
      // P as the second product's B operand: keys along k, rows along n
      uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float a = s[nt][2 * e], c = s[nt][2 * e + 1];
          const uint32_t hi = pack2_out<T>(a, c);
          const T* const hp = reinterpret_cast<const T*>(&hi);
          ph[nt][e] = transpose8(hi);
          pl[nt][e] = transpose8(pack2_out<T>(a - to_float(hp[0]), c - to_float(hp[1])));
        }
#pragma unroll
      for (int d0 = 0; d0 < D / 16; d0 += kAhead) {
        if (d0 > 0) {
#pragma unroll
          for (int d = 0; d < kAhead; ++d) ldsm4t(va[d], vs + v_row + (((2 * (d0 + d) + ((lane >> 3) & 1)) ^ v_key) << 4));
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
        for (int d = 0; d < kAhead; ++d)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma<T>(o[(d0 + d) * NT + nt], va[d], ph[nt][0], ph[nt][1]);
#pragma unroll
        for (int d = 0; d < kAhead; ++d)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma<T>(o[(d0 + d) * NT + nt], va[d], pl[nt][0], pl[nt][1]);
        if (apart) {
          for (int k = apart0; k < apart1; ++k) {
            const int src = (k & 7) * 4 + (lane & 3);
            const unsigned char* const row = st + (BK + key0 + k) * C::PITCH;
            const int ck = C::key(key0 + k);
            auto v_at = [&](int ch) { return to_float(reinterpret_cast<const T*>(row + (ch ^ ck) * 16)[lane >> 2]); };  // head dim 8 ch + lane / 4
            const int j = b.kb * BK + key0 + k;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                const float w = __shfl_sync(0xffffffffu, k < 8 ? s[nt][x] : s[nt][x + 2], src);
                if (j < limit[2 * nt + x]) {
#pragma unroll
                  for (int d = d0; d < d0 + kAhead; ++d) {
                    o[d * NT + nt][x] = fmaf(w, v_at(2 * d), o[d * NT + nt][x]);
                    o[d * NT + nt][x + 2] = fmaf(w, v_at(2 * d + 1), o[d * NT + nt][x + 2]);
                  }
                }
              }
          }
        }
      }
    }

    // ---- end of the unit, or of this CTA's part of it: the warps' sums are joined ----
    if (b.kb == nb - 1 || i == n_iter - 1) {
      const bool whole = unit_kb0 == 0 && b.kb == nb - 1;
      const int slot = 2 * blockIdx.x + (unit_kb0 == 0 ? 1 : 0);
      if (tid == 0 && !whole && unit_kb0 == 0) {
        // the unit's last block, on the line with its slots, and the piece that holds it
        const long long units = ((long long)b.seq * p.H_kv + h) * p.row_tiles + (b.hr >> 16) + 1;
        p.meta[blockIdx.x] = make_int4(b.seq, b.hr, (int)((first + i - b.kb + nb - 1 + units * kUnitCost) / piece.share), b.len);
      }
#pragma unroll
      for (int c = 0; c < 2 * NT; ++c) {
        l[c] += __shfl_xor_sync(0xffffffffu, l[c], 4);
        l[c] += __shfl_xor_sync(0xffffffffu, l[c], 8);
        l[c] += __shfl_xor_sync(0xffffffffu, l[c], 16);
      }
      if (lane < 4) {
#pragma unroll
        for (int c = 0; c < 2 * NT; ++c) join_ml[warp * C::ROWS_G + (c >> 1) * 8 + 2 * lane + (c & 1)] = make_float2(m[c], l[c]);
      }
      float* const join = reinterpret_cast<float*>(st);   // once all warps are through with the block
#pragma unroll
      for (int part = 0; part < RG * NT; ++part) {      // 8 rows of one row group at a time
        const int pg = part / NT, nt = part % NT;
        __syncthreads();
        if (rg == pg) {
          float* const mine = join + kw * 8 * C::MP;
          if constexpr (kFp32) {
            constexpr int DV = (D + 31) / 32;
#pragma unroll
            for (int r = 0; r < 8; ++r)
#pragma unroll
              for (int y = 0; y < DV; ++y) {
                const int d = D >= 128 ? (y / 4) * 128 + lane * 4 + (y & 3) : lane * DV + y;
                if (d < D) mine[r * C::MP + d] = o[r][y];
              }
          } else {
#pragma unroll
            for (int d = 0; d < D / 16; ++d)
#pragma unroll
              for (int x = 0; x < 4; ++x)
                mine[(2 * (lane & 3) + (x & 1)) * C::MP + d * 16 + (lane >> 2) + (x >> 1) * 8] = o[d * NT + nt][x];
          }
        }
        __syncthreads();
        constexpr int Q4 = D / 4;
        for (int e = tid; e < 8 * Q4; e += C::THREADS) {
          const int rr = e / Q4, d = (e % Q4) * 4;
          const int rt = part * 8 + rr;                 // row of the tile
          const int r = row0 + rt;
          if (r >= p.R) continue;
          float all = -INFINITY;
          float2 ml[KW];
#pragma unroll
          for (int w = 0; w < KW; ++w) {
            ml[w] = join_ml[(pg * KW + w) * C::ROWS_G + nt * 8 + rr];
            all = fmaxf(all, ml[w].x);
          }
          float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
          float ls = 0.f;
#pragma unroll
          for (int w = 0; w < KW; ++w) {
            if (ml[w].x == -INFINITY && ml[w].y == 0.f) continue;
            const float f = weight(ml[w].x, all);
            const float4 x = *reinterpret_cast<const float4*>(join + (w * 8 + rr) * C::MP + d);
            ls += f * ml[w].y;
            sum.x += f * x.x; sum.y += f * x.y; sum.z += f * x.z; sum.w += f * x.w;
          }
          if (whole) {
            write_row<T>(p, b.seq, h, r, b.len, D, d, sum, all, ls);
          } else {
            *reinterpret_cast<float4*>(p.part_o + ((int64_t)slot * C::ROWS + rt) * D + d) = sum;
            if (d == 0) p.part_ml[slot * C::ROWS + rt] = make_float2(all, ls);
          }
        }
      }
      __syncthreads();
    }
  }
}

// Joins the parts of a unit, in the order of the pieces: block (c, row) takes a row of the unit that begins in piece c and ends
// in a later one.  Groups of D / 4 threads take the parts in turn, several loads in flight each, and are summed in their own order.
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(256) combine_kernel(const DecodeParams p) {
  constexpr int Q4 = D / 4, GROUPS = 256 / Q4;
  constexpr int MOST = 512;                       // parts whose weights are held at a time
  __shared__ float wt[MOST];
  __shared__ float red[8], red_l[8];
  __shared__ float4 sums[GROUPS][Q4];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 u = p.meta[blockIdx.x];
  if (u.x < 0) return;
  const int tid = threadIdx.x;
  const int c0 = blockIdx.x, n = u.z - c0 + 1;
  const int h = u.y & 0xffff, rt = blockIdx.y, r = (u.y >> 16) * ROWS + rt;
  if (r >= p.R) return;
  auto part = [&](int c) { return (int64_t)(2 * (c0 + c) + (c == 0)) * ROWS + rt; };

  float all = -INFINITY;
  for (int c = tid; c < n; c += 256) all = fmaxf(all, __ldcg(&p.part_ml[part(c)]).x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, o));
  if ((tid & 31) == 0) red[tid >> 5] = all;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) all = fmaxf(all, red[w]);

  const int group = tid / Q4, q = tid % Q4;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  float ls = 0.f;
  for (int base = 0; base < n; base += MOST) {
    const int m = min(MOST, n - base);
    if (base > 0) __syncthreads();
    for (int c = tid; c < m; c += 256) {
      const float2 x = __ldcg(&p.part_ml[part(base + c)]);
      const float w = weight(x.x, all);           // (a part that saw nothing, or only -inf, weighs nothing)
      wt[c] = w;
      ls += w * x.y;
    }
    __syncthreads();
#pragma unroll 8
    for (int c = group; c < m; c += GROUPS) {
      const float w = wt[c];
      const float4 x = __ldcg(reinterpret_cast<const float4*>(p.part_o + part(base + c) * D + q * 4));
      sum.x += w * x.x; sum.y += w * x.y; sum.z += w * x.z; sum.w += w * x.w;
    }
  }
  sums[group][q] = sum;
  ls = warp_sum(ls);
  if ((tid & 31) == 0) red_l[tid >> 5] = ls;
  __syncthreads();
  if (tid >= Q4) return;
  sum = sums[0][tid];
#pragma unroll
  for (int g = 1; g < GROUPS; ++g) {
    const float4 x = sums[g][tid];
    sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
  }
  ls = red_l[0];
#pragma unroll
  for (int w = 1; w < 8; ++w) ls += red_l[w];
  write_row<T>(p, u.x, h, r, u.w, D, tid * 4, sum, all, ls);
}

// What a shape runs on: rows of a tile, CTAs, workspace.
struct Plan {
  int rows, row_tiles, ctas_per_sm, bk;
  int (*launch)(const DecodeParams&, int ctas, int min_share, bool splits, cudaStream_t);
};

template <typename C>
int launch_config(const DecodeParams& p, int ctas, int min_share, bool splits, cudaStream_t s) {
  static std::atomic<unsigned long long> set{0};  // a bit for each device
  int dev = 0;
  VAFA_CUDA_CHECK(cudaGetDevice(&dev));
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (!(set.load(std::memory_order_acquire) & bit) || !bit) {
    VAFA_CUDA_CHECK(cudaFuncSetAttribute(decode_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    set.fetch_or(bit, std::memory_order_release);
  }
  {
    LaunchScope scope(kKPagedDecode, s);
    decode_kernel<C><<<ctas, C::THREADS, C::kSmem, s>>>(p, min_share);
    VAFA_LAUNCH_CHECK("paged_decode_kernel");
  }
  if (!splits) return 0;
  LaunchScope scope(kKPagedCombine, s);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas, p.R < C::ROWS ? p.R : C::ROWS);
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  // its blocks may be made while the kernel above still runs; they wait for its end
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  VAFA_CUDA_CHECK(cudaLaunchKernelEx(&cfg, combine_kernel<typename C::T, C::D, C::ROWS>, p));
  return 0;
}

template <typename C>
Plan plan_of(int R) { return Plan{C::ROWS, (R + C::ROWS - 1) / C::ROWS, C::CTAS, C::BK, launch_config<C>}; }

// The tile of a shape: the fewest rows that hold the unit's, up to what the registers allow.
template <typename T, int D>
Plan plan_for(int R) {
  if constexpr (sizeof(T) == 4) {
    if (R <= 8) return plan_of<Config<T, D, 1, 1, 4>>(R);
    return plan_of<Config<T, D, 1, 2, 4>>(R);
  } else if constexpr (D == 256) {
    if (R <= 8) return plan_of<Config<T, D, 1, 1, 4>>(R);
    if (R <= 16) return plan_of<Config<T, D, 1, 2, 4>>(R);
    return plan_of<Config<T, D, 1, 4, 4>>(R);
  } else {
    if (R <= 8) return plan_of<Config<T, D, 1, 1, PD_KW>>(R);
    if (R <= 16) return plan_of<Config<T, D, 2, 1, 4>>(R);
    if (R <= 32) return plan_of<Config<T, D, 2, 2, 4>>(R);
    return plan_of<Config<T, D, 2, 4, 4>>(R);
  }
}

template <typename T>
Plan plan_by_dim(int D, int R) {
  switch (D) {
    case 16: return plan_for<T, 16>(R);
    case 32: return plan_for<T, 32>(R);
    case 64: return plan_for<T, 64>(R);
    case 128: return plan_for<T, 128>(R);
    default: return plan_for<T, 256>(R);
  }
}

Plan plan_bf16(int D, int R);
Plan plan_f16(int D, int R);
Plan plan_f32(int D, int R);

}  // namespace paged
}  // namespace vafa
