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
//  - each warp has its own keys of a block with its own maximum and sum (paged_decode_tiles.cuh), so that the loop has no exchange
//    between warps; they are joined once, at the unit's end.
// Measured: 128 caches of 8k to 32k keys, 8 heads of 128 in bf16 (10 GB) 1.41 to 1.50 ms, 6.7 to 7.1 TB/s (a copy moves 6.56); 64 caches of
// 1k to 16k keys, 32 query and 8 K/V heads (1.7 GB) 0.25 ms; 8 caches of up to 3k keys (59 MB) 18.5 us, 9 of them reading.
#pragma once
#include <atomic>

#include "paged_decode_tiles.cuh"
#include "profile.cuh"

namespace vafa {
namespace paged {

// How a shape is cut: RG groups of KW warps, a group's warps share out the keys of a block and have ROWS_G rows each; at most MOST CTAs an SM.
enum Kind { kNarrow, kWide, kFma4, kFma8 };  // (the last two: fp32, 4 or 8 rows a warp)
template <typename T_, int D_, Kind KIND_, int RG_, int KW_, int MOST_>
struct Config {
  using T = T_;
  static constexpr int D = D_, RG = RG_, KW = KW_;
  static constexpr Kind KIND = KIND_;
  static constexpr bool kFp32 = KIND == kFma4 || KIND == kFma8;
  static_assert(kFp32 == (sizeof(T) == 4), "fp32 has a tile of its own");
  static constexpr int NT = KIND == kWide ? 2 : 1;           // groups of 8 rows of a warp
  static constexpr int KPW = kFp32 ? (D >= 128 ? 8 : D == 64 ? 16 : 32) : KIND == kWide ? 64 / KW : D <= 64 ? 32 : 16;  // keys of a warp
  static constexpr int BK = KW * KPW;
  static constexpr int ROWS_G = KIND == kFma4 ? 4 : 8 * NT, ROWS = ROWS_G * RG;
  static constexpr int THREADS = 32 * KW * RG;
  static_assert(BK <= THREADS, "a thread looks up a key's place");
  static constexpr int VEC = 16 / (int)sizeof(T), CH = D / VEC;
  static_assert(THREADS % CH == 0, "a thread copies the same chunk of all its rows");
  // A row's 16-byte chunks are stored at chunk ^ key(row): the 8 rows that an ldmatrix tile reads at the same chunk then lie in
  // different banks without padding (fp32: so do the 64 bytes that 4 lanes read of each of two neighbouring rows).
  static constexpr int PITCH = D * (int)sizeof(T);
  static __device__ __forceinline__ int key(int row) {
    if constexpr (kFp32) return CH >= 8 ? (row & 1) * 4 : 0;
    else return (row / (CH < 8 ? 8 / CH : 1)) & ((CH < 8 ? CH : 8) - 1);
  }
  static constexpr int kStageBytes = (2 * BK + ROWS) * PITCH;
  static constexpr bool kQReg = KIND == kNarrow || (KIND == kWide && D <= 128);  // Q fragments stay in registers
  static constexpr int kQBytes = kQReg ? 0 : ROWS * PITCH;
  static constexpr int MP = KIND == kWide ? D + 8 : D + 4;                         // pitch of the join buffer, floats: 8 rows of each warp of a row group
  static constexpr int kJoinBytes = KW * 8 * MP * 4;
  static_assert(kJoinBytes <= kStageBytes, "the join buffer takes the place of a stage that has been read");
  static constexpr int kMlBytes = RG * KW * ROWS_G * 8;
  static constexpr int kPBytes = kFp32 ? RG * KW * (KPW + 2) * ROWS_G * 4 : 0;
  static constexpr int kBudget = 227 * 1024;
  static constexpr int kMaxStages = 6;
  // Places of keys are held for two blocks, those that are looked up before the loop in the stage that the loop fills first.
  static constexpr int row_slots(int s) { return (s - 1) * BK * 16 <= kStageBytes ? 2 : s + 1; }
  static constexpr int bytes_of(int s) { return s * kStageBytes + kQBytes + kMlBytes + kPBytes + row_slots(s) * BK * 16 + (s + 2) * 16 + 256; }
  static constexpr int fit(int ctas) {
    int s = kMaxStages;
    while (s > 1 && (bytes_of(s) + 1024) * ctas > kBudget + 1024) --s;
    return s;
  }
  static constexpr int CTAS = MOST_ >= 4 && fit(4) >= 2 ? 4 : MOST_ >= 3 && fit(3) >= 2 ? 3 : MOST_ >= 2 && fit(2) >= 2 ? 2 : 1;
  static constexpr int kRegisters = 65536 / (THREADS * CTAS);
  static constexpr int S = fit(CTAS);
  static constexpr int kInfo = S + 2;                      // slots of the ring of block descriptions
  static_assert(S >= 2, "no room for two stages");
  static constexpr int kSmem = bytes_of(S);
  using Tile = std::conditional_t<kFp32, Fp32Tile<Config>, std::conditional_t<KIND == kWide, WideTile<Config>, NarrowTile<Config>>>;
};

// A piece of the line of blocks: what a CTA needs to know to find its first block.  A unit costs more than its blocks (its
// queries, the join of the warps, the rows' way out), so the line that is cut has `kUnitCost` slots more in front of each
// unit's blocks; a piece that begins or ends among those begins or ends with the unit's first block.
// (32 caches of 7 to 7.2k keys, four tokens of 32 heads, 0 | 1 | 2 | 4 slots: 94 | 67 | 59 | 58 us; level on batches of one length)
constexpr int kUnitCost = 2;
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
__device__ void find_piece(const DecodeParams& p, Piece* out, long long* scan) {
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

__device__ __forceinline__ int page_of(const DecodeParams& p, int j) {
  return p.page_mul ? (int)(__umulhi((uint32_t)j, p.page_mul) >> p.page_shift) : j >> p.page_shift;
}

struct Block {  // a block of the line, as its ring slot describes it
  int seq, hr, kb, len;   // hr: K/V head, and row tile in the upper half
};

// Four dims of a row's sum of p v where P went into the product as two pieces and the sum is NaN although the weights are numbers: an infinite
// value gave inf - inf, or 0 inf where a piece is zero.  The values of keys [from, to) that are not finite decide, each with its whole
// weight, and where there is none NaN stays.  (64 caches of 4k to 8k keys, heads of 128, seven tokens of 8 grouped heads: 516 us without, 531 with
// this, 567 with a look over every block's values before the product; up to 16 rows level.  A thread walks over its keys until nothing
// more can change: 64 caches of 16k keys, 8 heads, whose last key alone is infinite or NaN in all dims 12 ms instead of 0.65, NaN everywhere 0.65.)
template <typename T, int D, typename Read, typename Write>
__device__ __forceinline__ void bad_values(const DecodeParams& p, int seq, int h, int r, int from, int to, int d, float m, Read sum, Write set) {
  const int t = r / p.g;
  const T* const q = reinterpret_cast<const T*>(p.q) + seq * p.q_seq + t * p.q_token + (h * p.g + r - t * p.g) * p.q_head;
  float now[4] = {0.f, 0.f, 0.f, 0.f};
  int found = 0, open = 0;  // dims that a value has been found for, dims that another one could change
#pragma unroll
  for (int x = 0; x < 4; ++x) open |= isnan(sum(x)) << x;
#pragma unroll 1
  for (int j = from; j < to && open; ++j) {
    const int row = page_of(p, j), page = p.table[seq * p.table_stride + row], slot = j - row * p.page_size;
    if (page < 0 || page >= p.num_pages) continue;
    const T* const v = reinterpret_cast<const T*>(p.v) + page * p.v_page + slot * p.v_slot + h * p.v_head + d;
    const uint2 raw = *reinterpret_cast<const uint2*>(v);
    if (!not_finite2<T>(raw.x) && !not_finite2<T>(raw.y)) continue;
    float w = 0.f;
    bool known = false;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float value = to_float(v[x]);
      if (isfinite(value) || !(open >> x & 1)) continue;
      if (!isnan(value) && !known) {
        const T* const k = reinterpret_cast<const T*>(p.k) + page * p.k_page + slot * p.k_slot + h * p.k_head;
        float s = 0.f;
#pragma unroll 8
        for (int i = 0; i < D; ++i) s = fmaf(to_float(q[i]), to_float(k[i]), s);
        w = exp2_approx(s * p.scale_log2 - m);
        known = true;
      }
      now[x] = fmaf(w, value, now[x]);  // (NaN whatever the weight)
      found |= 1 << x;
      if (isnan(now[x])) open &= ~(1 << x);
    }
  }
#pragma unroll
  for (int x = 0; x < 4; ++x)
    if (found >> x & 1) set(x, now[x]);
}

template <typename C>
__global__ void __launch_bounds__(C::THREADS, C::CTAS) decode_kernel(const DecodeParams p) {
  using T = typename C::T;
  constexpr int D = C::D, NT = C::NT, RG = C::RG, BK = C::BK, KW = C::KW, S = C::S;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ Piece piece;
  __shared__ volatile int missing;     // a page outside the cache has been met
  __shared__ long long scan[C::THREADS / 32];

  unsigned char* const stages = smem;
  unsigned char* at = smem + S * C::kStageBytes;
  unsigned char* const q_now = at;                     at += C::kQBytes;
  float2* const join_ml = reinterpret_cast<float2*>(at); at += C::kMlBytes;
  float* const p_all = reinterpret_cast<float*>(at);   at += C::kPBytes;
  at = smem + (((at - smem) + 15) & ~15);
  constexpr int kRowSlots = C::row_slots(S);
  longlong2* const row_at = reinterpret_cast<longlong2*>(at); at += kRowSlots * BK * 16;
  Block* const info = reinterpret_cast<Block*>(at);

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int kw = warp % KW, rg = warp / KW;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) missing = 0;
  find_piece<C>(p, &piece, scan);
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
  auto rows_of = [&](int i) { return row_at + i % kRowSlots * BK; };
  auto first_rows_of = [&](int i) {  // before the loop
    return kRowSlots == 2 && i < S - 1 ? reinterpret_cast<longlong2*>(stages + (S - 1) * C::kStageBytes) + i * BK : rows_of(i);
  };
  // a key's place in bytes from the head's first element; 0 for what lies behind the sequence, -1 for a page that is not there
  auto land = [&](const Lookup& x, int i, longlong2* rows) {
    if (tid == 0) info[i % C::kInfo] = x.b;
    longlong2 r = make_longlong2(0, 0);
    if (x.b.seq < p.n_seq && x.b.kb * BK + tid < x.b.len) {
      if (x.page >= 0 && x.page < p.num_pages) {
        r = make_longlong2((x.page * p.k_page + x.slot * p.k_slot) * (int)sizeof(T), (x.page * p.v_page + x.slot * p.v_slot) * (int)sizeof(T));
      } else {
        r = make_longlong2(-1, -1);
        missing = 1;
        report_error(p.status, kBadCacheIndex, kSiteDecode, x.b.seq);
      }
    }
    rows[tid] = r;
  };
  // copies block i (of this CTA) into its stage
  auto issue = [&](int i, const longlong2* places) {
    const Block b = info[i % C::kInfo];
    const longlong2* const rows = places + tid / C::CH;
    const int h = b.hr & 0xffff;
    unsigned char* const st = stages + (i % S) * C::kStageBytes;
    const char* const kh = reinterpret_cast<const char*>(reinterpret_cast<const T*>(p.k) + h * p.k_head) + tid % C::CH * 16;
    const char* const vh = reinterpret_cast<const char*>(reinterpret_cast<const T*>(p.v) + h * p.v_head) + tid % C::CH * 16;
    const uint32_t ks = smem_addr(st), vs = ks + BK * C::PITCH, qs = vs + BK * C::PITCH;
    constexpr int kRows = C::THREADS / C::CH;             // rows of a step: a thread has the same chunk of each of its rows
    const int here = b.len - b.kb * BK;                   // keys of the block
    auto copy = [&](auto all) {
#pragma unroll
      for (int x = 0; x < (BK + kRows - 1) / kRows; ++x) {
        const int row = x * kRows + tid / C::CH;
        if (BK % kRows != 0 && row >= BK) break;
        const longlong2 r = rows[x * kRows];
        const int to = row * C::PITCH + ((tid % C::CH) ^ C::key(row)) * 16;
        if (decltype(all)::value) {
          copy16(ks + to, kh + r.x, true);
          copy16(vs + to, vh + r.y, true);
        } else {  // zeros behind the sequence, and for pages that are not there
          const bool real = row < here && r.x >= 0;
          copy16(ks + to, kh + (real ? r.x : 0), real);
          copy16(vs + to, vh + (real ? r.y : 0), real);
        }
      }
    };
    if (here >= BK && !missing) copy(std::true_type{});
    else copy(std::false_type{});
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
    for (int i = 0; i < S; ++i) land(x[i], i, first_rows_of(i));
  }
  Lookup next;
  if (looks_up) {
    start(next);  // of block S
    walk();
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < S - 1; ++i) {
    if (i < n_iter) issue(i, first_rows_of(i));
    copy_commit();
  }

  typename C::Tile tile(Place{lane, kw, rg});
  int unit_kb0 = 0;                    // first block of the unit that this CTA has

  for (int i = 0; i < n_iter; ++i) {
    copy_wait<S - 2>();
    __syncthreads();
    if (i + S - 1 < n_iter) issue(i + S - 1, rows_of(i + S - 1));
    copy_commit();
    if (looks_up) {
      land(next, i + S, rows_of(i + S));
      start(next);
      walk();
    }
    const Block b = info[i % C::kInfo];
    unsigned char* const st = stages + (i % S) * C::kStageBytes;
    const int nb = blocks_of<BK>(b.len);
    const int h = b.hr & 0xffff, row0 = (b.hr >> 16) * C::ROWS;

    if (i == 0 || b.kb == 0) {
      unit_kb0 = b.kb;
      const unsigned char* q = st + 2 * BK * C::PITCH;
      if constexpr (!C::kQReg) {  // the stage goes, the queries stay
        for (int e = tid; e < C::ROWS * C::CH; e += C::THREADS)
          *reinterpret_cast<uint4*>(q_now + e * 16) = *reinterpret_cast<const uint4*>(q + e * 16);
        __syncthreads();
        q = q_now;
      }
      tile.begin(p, q, b.len, row0, p_all + warp * (C::KPW + 2) * C::ROWS_G);
    }
    BlockView view;
    view.k = st;
    view.v = st + BK * C::PITCH;
    view.first = b.kb * BK;
    view.len = b.len;
    view.every = b.len - p.T + 1;
    view.masked = (b.kb + 1) * BK > view.every;
    tile.block(p, view);

    // ---- end of the unit, or of this CTA's part of it: the warps' sums are joined ----
    if (b.kb == nb - 1 || i == n_iter - 1) {
      const bool whole = unit_kb0 == 0 && b.kb == nb - 1;
      const int slot = 2 * blockIdx.x + (unit_kb0 == 0 ? 1 : 0);
      if (tid == 0 && !whole && unit_kb0 == 0) {
        // the unit's last block, on the line with its slots, and the piece that holds it
        const long long units = ((long long)b.seq * p.H_kv + h) * p.row_tiles + (b.hr >> 16) + 1;
        p.meta[blockIdx.x] = make_int4(b.seq, b.hr, (int)((first + i - b.kb + nb - 1 + units * kUnitCost) / piece.share), b.len);
      }
      tile.stats(join_ml + warp * C::ROWS_G);
      bool bad = false;                                   // a sum that is NaN though its weights are numbers
      float* const join = reinterpret_cast<float*>(st);   // once all warps are through with the block
#pragma unroll
      for (int part = 0; part < RG * NT; ++part) {      // 8 rows of one row group at a time
        const int pg = part / NT, nt = part % NT;
        __syncthreads();
        if (rg == pg) tile.rows(join + kw * 8 * C::MP, nt);
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
          if constexpr (!C::kFp32) bad |= isnan(sum.x + sum.y + sum.z + sum.w) && !isnan(ls);
          if (whole) {
            write_row<T>(p, b.seq, h, r, b.len, D, d, sum, all, ls);
          } else {
            *reinterpret_cast<float4*>(p.part_o + ((int64_t)slot * C::ROWS + rt) * D + d) = sum;
            if (d == 0) p.part_ml[slot * C::ROWS + rt] = make_float2(all, ls);
          }
        }
      }
      if constexpr (C::kFp32) {
        __syncthreads();
      } else if (__syncthreads_or(bad)) {
        // which of the sums these are is in what has been written and in the warps' statistics
        for (int e = tid; e < C::ROWS * (D / 4); e += C::THREADS) {
          const int rt = e / (D / 4), d = e % (D / 4) * 4, r = row0 + rt;
          if (r >= p.R) break;
          float all = -INFINITY, ls = 0.f;
          for (int w = 0; w < KW; ++w) all = fmaxf(all, join_ml[(rt / C::ROWS_G * KW + w) * C::ROWS_G + rt % C::ROWS_G].x);
          for (int w = 0; w < KW; ++w) {
            const float2 ml = join_ml[(rt / C::ROWS_G * KW + w) * C::ROWS_G + rt % C::ROWS_G];
            ls += (ml.x == -INFINITY && ml.y == 0.f) ? 0.f : weight(ml.x, all) * ml.y;
          }
          if (isnan(ls)) continue;
          const int t = r / p.g;
          T* const o = reinterpret_cast<T*>(p.o) + (((int64_t)b.seq * p.T + t) * p.H + h * p.g + r - t * p.g) * D + d;
          float* const part = p.part_o + ((int64_t)slot * C::ROWS + rt) * D + d;
          bad_values<T, D>(p, b.seq, h, r, unit_kb0 * BK, min((b.kb + 1) * BK, row_limit(p, b.len, r)), d, all,
                           [&](int x) { return whole ? to_float(o[x]) : part[x]; },
                           [&](int x, float value) { if (whole) o[x] = from_float<T>(value); else part[x] = value; });
        }
      }
    }
  }
}

// Joins the parts of a unit, in the order of the pieces: blocks (c, *) take the unit that begins in piece c and ends in a later one.
// A unit of few parts is joined row by row, D / 4 threads a row; the rows of one in many pieces (few units, long ones) are each
// joined by a whole block, whose groups of D / 4 threads take the parts in turn and are summed in their own order.
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(256) combine_kernel(const DecodeParams p) {
  constexpr int Q4 = D / 4, GROUPS = 256 / Q4;
  constexpr int FEW = 8, MOST = 256;              // parts that a thread takes alone; parts whose weights are held at a time
  __shared__ float wt[MOST];
  __shared__ float red[8], red_l[8];
  __shared__ float4 sums[GROUPS][Q4];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 u = p.meta[blockIdx.x];
  if (u.x < 0) return;
  const int tid = threadIdx.x, group = tid / Q4, q = tid % Q4;
  const int c0 = blockIdx.x, n = u.z - c0 + 1;
  const int h = u.y & 0xffff, row0 = (u.y >> 16) * ROWS, rows = min(ROWS, p.R - row0);
  auto part = [&](int c, int rt) { return (int64_t)(2 * (c0 + c) + (c == 0)) * ROWS + rt; };

  if (n <= FEW) {
    for (int rt = blockIdx.y * GROUPS + group; rt < rows; rt += gridDim.y * GROUPS) {
      float2 ml[FEW];
      float4 x[FEW];
#pragma unroll
      for (int c = 0; c < FEW; ++c)
        if (c < n) {
          ml[c] = __ldcg(&p.part_ml[part(c, rt)]);
          x[c] = __ldcg(reinterpret_cast<const float4*>(p.part_o + part(c, rt) * D + q * 4));
        }
      float all = -INFINITY;
#pragma unroll
      for (int c = 0; c < FEW; ++c)
        if (c < n) all = fmaxf(all, ml[c].x);
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      float ls = 0.f;
#pragma unroll
      for (int c = 0; c < FEW; ++c)
        if (c < n) {
          const float w = weight(ml[c].x, all);   // (a part that saw nothing, or only -inf, weighs nothing)
          ls += w * ml[c].y;
          sum.x += w * x[c].x; sum.y += w * x[c].y; sum.z += w * x[c].z; sum.w += w * x[c].w;
        }
      write_row<T>(p, u.x, h, row0 + rt, u.w, D, q * 4, sum, all, ls);
    }
    return;
  }

  for (int rt = blockIdx.y; rt < rows; rt += gridDim.y) {
    float all = -INFINITY;
    for (int c = tid; c < n; c += 256) all = fmaxf(all, __ldcg(&p.part_ml[part(c, rt)]).x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, o));
    if ((tid & 31) == 0) red[tid >> 5] = all;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) all = fmaxf(all, red[w]);

    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    float ls = 0.f;
    for (int base = 0; base < n; base += MOST) {
      const int m = min(MOST, n - base);
      if (base > 0) __syncthreads();
      if (tid < m) {
        const float2 x = __ldcg(&p.part_ml[part(base + tid, rt)]);
        const float w = weight(x.x, all);
        wt[tid] = w;
        ls += w * x.y;
      }
      __syncthreads();
#pragma unroll 8
      for (int c = group; c < m; c += GROUPS) {
        const float w = wt[c];
        const float4 x = __ldcg(reinterpret_cast<const float4*>(p.part_o + part(base + c, rt) * D + q * 4));
        sum.x += w * x.x; sum.y += w * x.y; sum.z += w * x.z; sum.w += w * x.w;
      }
    }
    sums[group][q] = sum;
    ls = warp_sum(ls);
    if ((tid & 31) == 0) red_l[tid >> 5] = ls;
    __syncthreads();
    if (tid < Q4) {
      sum = sums[0][tid];
#pragma unroll
      for (int g = 1; g < GROUPS; ++g) {
        const float4 x = sums[g][tid];
        sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
      }
      ls = red_l[0];
#pragma unroll
      for (int w = 1; w < 8; ++w) ls += red_l[w];
      write_row<T>(p, u.x, h, row0 + rt, u.w, D, tid * 4, sum, all, ls);
    }
    __syncthreads();
  }
}

// What a shape runs on: rows of a tile, CTAs, workspace.
struct Plan {
  int rows, row_tiles, ctas_per_sm, bk;
  int (*launch)(const DecodeParams&, int ctas, bool splits, cudaStream_t);
};

template <typename C>
int launch_config(const DecodeParams& p, int ctas, bool splits, cudaStream_t s) {
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
    decode_kernel<C><<<ctas, C::THREADS, C::kSmem, s>>>(p);
    VAFA_LAUNCH_CHECK("paged_decode_kernel");
  }
  if (!splits) return 0;
  LaunchScope scope(kKPagedCombine, s);
  cudaLaunchConfig_t cfg{};
  // a block for 256 x 4 values of a unit, or one for each row where units are in many parts
  const int rows = p.R < C::ROWS ? p.R : C::ROWS;
  const bool many = (long long)p.n_seq * p.H_kv * p.row_tiles * 6 < ctas;
  cfg.gridDim = dim3(ctas, many ? rows : (rows * C::D / 4 + 255) / 256);
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

// The tile of a shape, by the rows of its units and the head dim.  What decides is how many warps there are to hide latencies, then how
// often an SM reads a block from shared memory.  64 caches of 4k to 8k keys with 8 K/V heads of 128, us:
//   up to 8 rows     narrow; 1 | 2 | 3 CTAs an SM (128 caches of 8k to 32k keys) 2782 | 1585 | 1427
//   up to 16         wide, 4 warps on a block, 3 CTAs: 256; two 264, one 442; two warps on a block 351; narrow with two column tiles 292
//   up to 32         wide, 2 row groups of 2 warps, 2 CTAs: 345; (of the first version) 361; one CTA 592; 4 warps a group 441, one 532
//   up to 64         wide, 4 row groups of 1 warp, 2 CTAs: 531; (of the first version) 534; of 2 warps, one CTA 636; of 4 warps 1165
//   heads of 256     O takes twice the registers: narrow with two row groups to 16 rows, 287 (wide 376), wide beyond (28 rows 387)
//   fp32             4 rows a warp where units have no more, 3 CTAs: 507; 8 rows 877 (two groups of 4: 851, but no gain with more rows)
template <typename T, int D>
Plan plan_for(int R) {
  if constexpr (sizeof(T) == 4) {
    if (R <= 4) return plan_of<Config<T, D, kFma4, 1, 4, 3>>(R);
    if (R <= 8) return plan_of<Config<T, D, kFma8, 1, 4, 3>>(R);
    return plan_of<Config<T, D, kFma8, 2, 4, 2>>(R);
  } else {
    if (R <= 8) return plan_of<Config<T, D, kNarrow, 1, 4, 3>>(R);  // (one CTA at heads of 256: no room for two)
    if constexpr (D == 256) {
      if (R <= 16) return plan_of<Config<T, D, kNarrow, 2, 4, 1>>(R);
      return plan_of<Config<T, D, kWide, 2, 4, 1>>(R);
    } else {
      if (R <= 16) return plan_of<Config<T, D, kWide, 1, 4, 3>>(R);
      if (R <= 32) return plan_of<Config<T, D, kWide, 2, 2, D <= 64 ? 3 : 2>>(R);
      return plan_of<Config<T, D, kWide, 4, 1, D <= 64 ? 3 : 2>>(R);
    }
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
