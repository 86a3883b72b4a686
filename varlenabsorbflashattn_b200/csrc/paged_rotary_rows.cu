// The rotation of long batches: token rows go through shared memory.
//
// The work per byte is a few instructions, so what counts is how many bytes are on their way.  Held in registers (paged_rotary.cu)
// they are 30 to 60 KB an SM, and a block's start, look-ups and loads follow one another: 4.1 TB/s.  Here a warp looks positions
// and places up and sends for the rows and angles of a tile of tokens by bulk copies, four tiles ahead (eight, where 216 KB hold as many: 27 KB
// or less); sixteen warps rotate them in place in shared memory, in groups that take turns; another warp sends them to the outputs, or to the cache's slots, by bulk
// copies.  Values that only move (v) are not touched by a thread.  151 k tokens of 40 heads of 128 (3.1 GB in and out): 0.49 ms,
// 6.3 TB/s, 96 % of a plain copy; into a cache of pages of 16 (18 k tokens, 0.45 GB) 75 us, 91 %.
#include <atomic>
#include <type_traits>

#include "paged_rotary.cuh"
#include "sm100_ptx.cuh"

namespace vafa {
namespace rotary {
namespace {

// groups of warps, each with every kGroups-th tile: a tile's waits and its fence are as long as its arithmetic
constexpr int kGroups = 4, kCompute = 32 * 4, kComputeWarps = kGroups * 4, kThreads = 32 * kComputeWarps + 64;
constexpr int kMaxStages = 8, kMaxTokens = 32;
constexpr int kSite = 913;
static_assert(kMaxStages == 8 && kGroups == 4, "4 or 8 stages: one or three tiles on their way out");

struct Rows {
  int tokens, stages, tiles;        // tokens of a tile, tiles in flight, tiles in all
  // a tile is the rows of its tokens for one group after the other, then their cosines, then their sines
  int tile_bytes;
  int row_bytes[3], at[3];          // bytes of a group's part of a token (0: no such group), and where the group begins in a tile
  int angle_at, angle_bytes;        // where the cosines begin, bytes of a token's (0: read from the table in HBM)
  int turned[2];                    // heads of the first two groups that rotate
  int chunks;                       // chunks of VW pairs of a head
  int merged;                       // groups whose tokens lie side by side in their source: one copy a tile
  int wait_limit;
};

struct Control {
  uint64_t full[kMaxStages], done[kMaxStages], empty[kMaxStages];
  int4 info[kMaxStages][kMaxTokens];  // fate, page, slot, position
  int abort_flag;
  int wait_limit;                   // (read by the bounded waits as abort_flag[1])
};

__device__ __forceinline__ void bulk_store(void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
}

template <typename T, int VW, bool INTER, bool APPEND>
__global__ void __launch_bounds__(kThreads, 1) rows_kernel(const Params p, const Rows w) {
  using namespace ptx;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ Control ctl;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* const abort_flag = &ctl.abort_flag;
  if (tid == 0) {
    ctl.abort_flag = 0;
    ctl.wait_limit = w.wait_limit;
    for (int i = 0; i < w.stages; ++i) {
      mbar_init(smem_u32(&ctl.full[i]), 32);
      mbar_init(smem_u32(&ctl.done[i]), kCompute);
      mbar_init(smem_u32(&ctl.empty[i]), 1);
    }
    fence_barrier_init();
  }
  __syncthreads();
  int stage = 0, phase = 0;
  auto advance = [&](int n = 1) {  // (n <= stages, which are a multiple of the groups)
    stage += n;
    if (stage >= w.stages) {
      stage -= w.stages;
      phase ^= 1;
    }
  };

  if (warp == kComputeWarps) {
    // ---- looks the tokens up and sends for their rows: a lane a token, of as many tiles as 32 lanes hold (the look-up, a chain of
    // dependent reads, is as long as several tiles take) ----
    const int per_batch = 32 / w.tokens;
    const int of_batch = lane / w.tokens, token = lane - of_batch * w.tokens;
    const uint32_t tile_lanes = (w.tokens < 32 ? (1u << w.tokens) - 1 : 0xffffffffu) << (of_batch < per_batch ? of_batch * w.tokens : 0);
    int sent = 0;
    bool ok = true;
    for (int64_t batch = blockIdx.x; ok && batch < w.tiles; batch += (int64_t)per_batch * gridDim.x) {
      const int64_t my_tile = batch + (int64_t)of_batch * gridDim.x, t = my_tile * w.tokens + token;
      const bool mine = of_batch < per_batch && my_tile < w.tiles && t < p.total;
      int pos = 0, page = 0, slot = 0;
      Fate fate = kDone;
      if (mine) fate = place_of<APPEND>(p, (int)t, true, &pos, &page, &slot);
      // angles of neighbouring positions are one copy: the first token of a run sends for all of them
      const bool turns = mine && fate == kDone && w.angle_bytes > 0;
      const int before = __shfl_up_sync(0xffffffffu, turns ? pos : -2, 1);
      const bool leads = !turns || token == 0 || pos != before + 1;
      const uint32_t leaders = (__ballot_sync(0xffffffffu, leads) & tile_lanes) >> lane >> 1;
      const int run = !turns || !leads ? 0 : leaders ? __ffs(leaders) : w.tokens - token;
      const int rows = mine && token == 0 ? (int)(p.total - t < w.tokens ? p.total - t : w.tokens) : 0;  // of the tile, for its first lane
      for (int i = 0; i < per_batch && batch + (int64_t)i * gridDim.x < w.tiles; ++i, ++sent) {
        ok = mbar_wait_warp(smem_u32(&ctl.empty[stage]), phase ^ 1, abort_flag);  // one answer: the lanes meet again in the next batch
        if (!ok) break;
        const uint32_t bar = smem_u32(&ctl.full[stage]);
        if (mine && of_batch == i) {
          ctl.info[stage][token] = make_int4(fate, page, slot, pos);
          uint32_t bytes = 2 * run * w.angle_bytes;
#pragma unroll
          for (int g = 0; g < 3; ++g) bytes += ((w.merged >> g) & 1 ? rows : 1) * w.row_bytes[g];
          mbar_expect_tx(bar, bytes);
          const uint32_t dst = smem_u32(smem) + stage * w.tile_bytes;
#pragma unroll
          for (int g = 0; g < 3; ++g) {
            const int n = (w.merged >> g) & 1 ? rows : 1;
            if (w.row_bytes[g] > 0 && n > 0)
              bulk_load_1d(dst + w.at[g] + token * w.row_bytes[g], reinterpret_cast<const T*>(p.g[g].src) + t * p.g[g].token_stride,
                           n * w.row_bytes[g], bar);
          }
          if (run > 0) {
            const uint32_t to = dst + w.angle_at + token * w.angle_bytes;
            bulk_load_1d(to, p.cos + (int64_t)pos * (p.R / 2), run * w.angle_bytes, bar);
            bulk_load_1d(to + w.tokens * w.angle_bytes, p.sin + (int64_t)pos * (p.R / 2), run * w.angle_bytes, bar);
          }
        } else {
          mbar_arrive(bar);
        }
        advance();
      }
    }
    // what is still on its way lands before the block ends, also when another role has given up
    for (int i = sent > w.stages ? sent - w.stages : 0; i < sent; ++i)
      for (int polls = 0; polls < (1 << 20) && !mbar_test_wait(smem_u32(&ctl.full[i % w.stages]), (i / w.stages) & 1); ++polls) {}
  } else if (warp > kComputeWarps) {
    // ---- sends the rows off: a lane a token.  As many tiles as half the stages are on their way out before the first one's buffer
    // is asked back ----
    const int behind = w.stages / 2 - 1;
    int sent = 0;
    for (int64_t tile = blockIdx.x; tile < w.tiles; tile += gridDim.x, ++sent) {
      if (!mbar_wait_warp(smem_u32(&ctl.done[stage]), phase, abort_flag)) break;
      const int64_t t = tile * w.tokens + lane;
      if (lane < w.tokens && t < p.total) {
        const int4 info = ctl.info[stage][lane];
        const int rows = (int)(p.total - t < w.tokens ? p.total - t : w.tokens);
        const uint32_t base = smem_u32(smem) + stage * w.tile_bytes;
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          if (w.row_bytes[i] == 0) continue;
          const HeadGroup& g = p.g[i];
          const uint32_t src = base + w.at[i] + lane * w.row_bytes[i];
          if (!g.cached) {  // a packed output: the tile's rows lie side by side
            if (lane == 0) bulk_store(reinterpret_cast<T*>(g.dst) + t * g.page_stride, src, rows * w.row_bytes[i]);
          } else if (info.x == kDone) {
            T* const dst = reinterpret_cast<T*>(g.dst) + info.y * g.page_stride + info.z * g.slot_stride;
            if (g.dst_head_stride == p.D) {
              bulk_store(dst, src, w.row_bytes[i]);
            } else {
              const uint32_t head = p.D * sizeof(T);
              for (uint32_t x = 0; x * head < (uint32_t)w.row_bytes[i]; ++x) bulk_store(dst + x * g.dst_head_stride, src + x * head, head);
            }
          }
        }
      }
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      if (sent >= behind) {
        if (behind == 3) asm volatile("cp.async.bulk.wait_group.read 3;" ::: "memory");
        else asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
        __syncwarp();
        const int freed = stage - behind;
        if (lane == 0) mbar_arrive(smem_u32(&ctl.empty[freed < 0 ? freed + w.stages : freed]));
      }
      advance();
    }
    bulk_store_wait();
  } else {
    // ---- rotates in place: the threads of a tile are shared out among its tokens, a thread keeps its pairs' angles over all heads ----
    const int per_token = kCompute / w.tokens;
    const int group = tid / kCompute, in_group = tid - group * kCompute;
    const int token = in_group / per_token, in_token = in_group - token * per_token;
    const int chunks = w.chunks, lanes = chunks ? per_token / chunks : 0;
    const int hl = chunks ? in_token / chunks : 0, c = in_token - hl * chunks;
    const int d0 = INTER ? 2 * c * VW : c * VW, d1 = INTER ? d0 + VW : p.R / 2 + c * VW;
    advance(group);
    for (int64_t tile = blockIdx.x + (int64_t)group * gridDim.x; tile < w.tiles; tile += kGroups * gridDim.x) {
      if (!mbar_wait(smem_u32(&ctl.full[stage]), phase, abort_flag)) break;
      const int64_t t = tile * w.tokens + token;
      if (token < w.tokens && t < p.total) {
        const int4 info = ctl.info[stage][token];
        unsigned char* const base = smem + stage * w.tile_bytes;
        if (info.x != kDone) {
          const uint32_t nan = sizeof(T) == 4 ? 0x7fc00000u : std::is_same<T, __half>::value ? 0x7e007e00u : 0x7fc07fc0u;
          const uint32_t f = info.x == kZeros ? 0u : nan;
#pragma unroll
          for (int g = 0; g < 3; ++g)
            if (w.row_bytes[g] > 0 && !p.g[g].cached)
              for (int x = in_token * 16; x < w.row_bytes[g]; x += per_token * 16)
                *reinterpret_cast<uint4*>(base + w.at[g] + token * w.row_bytes[g] + x) = make_uint4(f, f, f, f);
        } else if (hl < lanes) {
          float cs[VW], sn[VW];
          if (w.angle_bytes) {
            const float* const a = reinterpret_cast<const float*>(base + w.angle_at + token * w.angle_bytes) + c * VW;
            load_angles<VW>(a, a + w.tokens * (p.R / 2), p.sign, cs, sn);
          } else {
            const int64_t at = (int64_t)info.w * (p.R / 2) + c * VW;
            load_angles<VW>(p.cos + at, p.sin + at, p.sign, cs, sn);
          }
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            T* const row = reinterpret_cast<T*>(base + w.at[g] + token * w.row_bytes[g]);
            // (the second group's heads go on where the first one's end)
            int h = g == 0 || w.turned[0] == 0 ? hl : hl - w.turned[0] % lanes;
            if (h < 0) h += lanes;
#pragma unroll 4
            for (; h < w.turned[g]; h += lanes) {
              Vec<T, VW>* const px = reinterpret_cast<Vec<T, VW>*>(row + h * p.D + d0);
              Vec<T, VW>* const py = reinterpret_cast<Vec<T, VW>*>(row + h * p.D + d1);
              Vec<T, VW> x = *px, y = *py;
              rotate<T, VW, INTER>(x, y, cs, sn);
              *px = x;
              *py = y;
            }
          }
        }
      }
      fence_proxy_async();
      mbar_arrive(smem_u32(&ctl.done[stage]));
      advance(kGroups);
    }
  }
  __syncthreads();
  if (tid == 0 && ctl.abort_flag != 0) report_error(p.status, 1, kSite, blockIdx.x);
}

template <typename T, int VW, bool INTER, bool APPEND>
int launch_one(const Params& p, const Rows& w, int blocks, int smem, cudaStream_t s) {
  static std::atomic<unsigned long long> set{0};  // a bit for each device
  int dev = 0;
  VAFA_CUDA_CHECK(cudaGetDevice(&dev));
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (!(set.load(std::memory_order_acquire) & bit) || !bit) {
    VAFA_CUDA_CHECK(cudaFuncSetAttribute(rows_kernel<T, VW, INTER, APPEND>, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024));
    set.fetch_or(bit, std::memory_order_release);
  }
  LaunchScope scope(kKRotaryRows, s);
  rows_kernel<T, VW, INTER, APPEND><<<blocks, kThreads, smem, s>>>(p, w);
  VAFA_LAUNCH_CHECK("rotary rows_kernel");
  return 0;
}

template <typename T, int VW>
int launch_width(const Params& p, const Rows& w, bool inter, bool append, int blocks, int smem, cudaStream_t s) {
  if (append) return inter ? launch_one<T, VW, true, true>(p, w, blocks, smem, s) : launch_one<T, VW, false, true>(p, w, blocks, smem, s);
  return inter ? launch_one<T, VW, true, false>(p, w, blocks, smem, s) : launch_one<T, VW, false, false>(p, w, blocks, smem, s);
}

template <typename T>
int launch_type(int vw, const Params& p, const Rows& w, bool inter, bool append, int blocks, int smem, cudaStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (vw == 8) return launch_width<T, 8>(p, w, inter, append, blocks, smem, s);
  }
  if (vw == 4) return launch_width<T, 4>(p, w, inter, append, blocks, smem, s);
  if (vw == 2) return launch_width<T, 2>(p, w, inter, append, blocks, smem, s);
  return launch_width<T, 1>(p, w, inter, append, blocks, smem, s);
}

}  // namespace

int launch_rows(Params& p, int vw, int dtype, bool inter, bool append, cudaStream_t s) {
  const int es = elem_size(dtype);
  // whole token rows that a bulk copy can take: heads side by side, addresses and sizes multiples of 16 bytes
  Rows w{};
  int64_t bytes = 0;
  bool turns = false;
  for (int i = 0; i < p.n_groups; ++i) {
    const HeadGroup& g = p.g[i];
    const int n = (i + 1 < p.n_groups ? p.g[i + 1].first : p.heads) - g.first;
    if ((n > 1 && g.head_stride != p.D) || ((uintptr_t)g.src | (uintptr_t)g.dst) % 16 ||
        ((g.token_stride | g.page_stride | g.slot_stride) * es) % 16 || (n > 1 && (g.dst_head_stride * es) % 16))
      return 1;
    if ((int64_t)n * p.D * es > 48 * 1024) return 1;
    w.row_bytes[i] = n * p.D * es;
    bytes += w.row_bytes[i];
    if (g.token_stride == (int64_t)n * p.D) w.merged |= 1 << i;
    if (g.rotate && i < 2) {
      w.turned[i] = n;
      turns = true;
    }
  }
  // From 10 MB on: below, the other kernel's one short chain is as fast (here | there: 4 000 tokens of 2 KB 7.2 | 6.5 us, 1600 of
  // 10 KB 7.9 | 8.8).  Not for tokens so short that the bookkeeping of 32 of them outweighs their bytes (256 000 of 256 bytes 68 | 52 us,
  // 64 000 of 2 KB 52 | 97), nor for rows of which four tiles do not fit.
  if (bytes < 1024 || bytes > 48 * 1024 || bytes * p.total < (10 << 20)) return 1;
  if (turns && (p.R * 2) % 16 == 0 && ((uintptr_t)p.cos | (uintptr_t)p.sin) % 16 == 0) w.angle_bytes = p.R * 2;
  const int token_bytes = (int)bytes + 2 * w.angle_bytes;
  w.chunks = turns ? p.R / (2 * vw) : 0;
  // (tiles of 40 KB | 20 KB: 151 k tokens of 10 KB 484 | 601 us, 27 k of them 90 | 108, 64 k of 2 KB 52 | 49)
  w.tokens = 40 * 1024 / token_bytes;
  const int most = w.chunks ? kCompute / w.chunks : kMaxTokens;
  if (w.tokens > most) w.tokens = most;
  if (w.tokens > kMaxTokens) w.tokens = kMaxTokens;
  if (w.tokens < 1) w.tokens = 1;
  for (int i = 0, at = 0; i < 3; ++i) {
    w.at[i] = at;
    at += w.tokens * w.row_bytes[i];
    w.angle_at = at;
  }
  w.tile_bytes = w.tokens * token_bytes;
  w.stages = 216 * 1024 / w.tile_bytes;
  if (w.stages > kMaxStages) w.stages = kMaxStages;
  // a stage belongs to one group (stages a multiple of the groups): a group that waited on a stage whose last tile was another
  // group's could take the end of the phase before that for the end of its own
  w.stages -= w.stages % kGroups;
  if (w.stages < kGroups) return 1;
  w.tiles = (int)(((int64_t)p.total + w.tokens - 1) / w.tokens);
  w.wait_limit = wait_limit_units();
  const int blocks = w.tiles < 148 ? w.tiles : 148, smem = w.stages * w.tile_bytes;
  if (dtype == VAFA_F32) return launch_type<float>(vw, p, w, inter, append, blocks, smem, s);
  if (dtype == VAFA_BF16) return launch_type<__nv_bfloat16>(vw, p, w, inter, append, blocks, smem, s);
  return launch_type<__half>(vw, p, w, inter, append, blocks, smem, s);
}

}  // namespace rotary
}  // namespace vafa
