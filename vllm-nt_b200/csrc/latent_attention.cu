// Latent attention over the paged latent cache (the absorbed form): every head of a token reads
// the same cached row c_j = [latent (512) | rotary key (64)],
//   s_j = scale * (q_latent . latent_j + q_rope . key_j),  out = sum_j softmax(s)_j latent_j,
// so a row is both key and value and is read from HBM once for all heads.  Query i of a
// sequence with q_len queries sits at position ctx - q_len + i and sees keys up to it.
//
// Work.  Query rows (token, head) of a sequence form groups of at most 64 rows: up to 64 heads
// of one token, or several tokens' heads when there are fewer.  An item is one group of one
// sequence, cut into tiles of 64 cached tokens; the tiles of all items, in order, are dealt to
// one CTA per SM in equal runs, so ragged batches balance and a long context with few rows is
// split over the GPU.  A run that starts or ends inside an item leaves that item's share
// (normalised output and log2 of the sum, fp32) in the workspace and a second kernel joins
// the shares.  When a sequence has several groups (up to kMaxTeams), CTA c takes group
// c % groups only: neighbours read the same tiles at the same time, the second from L2.
//
// One tile, 256 threads:
//   warp 0     TMA: the item's queries (9 chunks of 64 columns), then units of 16 cached tokens
//              into a ring of 8.  A unit is one copy of a 5-D box (64 columns, 8 tokens, 9 chunks,
//              2 groups of 8 tokens): whole rows are asked for together, and they land as the
//              1024-byte swizzled atoms that the MMAs read, [8-token group][chunk].
//   warp 1     S = Q C^T on tcgen05 (M = 64: rows past the group's are whatever shared memory
//              holds, and their lanes are never used; N = 64 tokens), two S buffers.
//   warp 2     O^T += C^T P^T: the cached rows as the MN-major A operand (M = 128 latent
//              columns, four times), P [rows, tokens] as B.  O^T takes 4 x rows TMEM columns
//              where O would need all 512, which leaves room for S and lets the tile that S
//              was made from be used as it lies.  A unit is free after its 16-token step.
//   warps 4-7  softmax: a warp the 16 rows of its TMEM lanes, four lanes a row, so a row's
//              maximum is two shuffles; refreshed only when it grows by over 2^8 (O^T is
//              rescaled then); and the output.
// The issuing warps stay converged and elect the lane for each instruction: descriptors then live
// in uniform registers (from a branch on one lane an MMA took 52 cycles to issue, so 48).
//
// Bound: HBM for a few rows (96 ragged contexts up to 8192, 16 heads: 99 us, 4.6 TB/s, a tile every
// 3470 cycles where its bytes need 3070).  With 64 rows the MMAs' operands take 2560 cycles of
// shared memory a tile, and the chain S, softmax, P, O^T through a ring of two tiles 3700 (32 contexts
// of 16384, 128 heads: 226 us; 251 us where calls follow each other for long, at the power limit's clock).
#include <algorithm>

#include "common.cuh"
#include "tcgen05.cuh"

namespace ntb200 {
namespace {

constexpr int kLatent = 512;
constexpr int kRope = 64;
constexpr int kChunks = (kLatent + kRope) / 64;  // 64-column chunks of a row; the last is rotary
constexpr int kTile = 64;                        // cached tokens a tile
constexpr int kUnit = 16;                        // cached tokens a copy, and an O^T step
constexpr int kGroupBytes = kChunks * 1024;      // 8 tokens: one 1024-byte atom a chunk
constexpr int kUnitBytes = 2 * kGroupBytes;
constexpr int kTileUnits = kTile / kUnit;
constexpr int kRing = 2 * kTileUnits;            // units
constexpr int kMTiles = kLatent / 128;           // M = 128 products that make up O^T
constexpr int kMaxRows = 64;                     // query rows a group
constexpr int kFirstSmWarp = 4;
constexpr int kSmThreads = 128;
constexpr int kThreads = 32 * kFirstSmWarp + kSmThreads;
constexpr int kMaxTeams = 8;
constexpr int kMaxCtas = 256;                    // one an SM
constexpr float kRescaleLog2 = 8.0f;

template <int N>
struct Layout {
  static constexpr int kQBufs = N == 64 ? 1 : 2;
  static constexpr int kQBytes = kChunks * N * 128;
  static constexpr int kQ = 0;
  static constexpr int kKv = kQ + kQBufs * kQBytes;
  static constexpr int kP = kKv + kRing * kUnitBytes;
  static constexpr int kRowF = kP + N * 128;           // [64] floats: a row's rescale, then 1 / sum
  static constexpr int kRowAt = kRowF + kMaxRows * 4;  // [64] int64: where a row's output goes
  static constexpr int kBars = kRowAt + kMaxRows * 8;  // mbarriers
  static constexpr int kQFull = 0, kQEmpty = kQFull + kQBufs, kFull = kQEmpty + kQBufs, kEmpty = kFull + kRing,
                       kSFull = kEmpty + kRing, kSFree = kSFull + 2, kPFull = kSFree + 2, kPvDone = kPFull + 1,
                       kOFree = kPvDone + 1, kMmaDone = kOFree + 1, kNumBars = kMmaDone + 1;
  static constexpr int kStart = kBars + 8 * kNumBars;  // the run's first tile, TMEM base, scan scratch
  static constexpr int kBytes = kStart + 32 + 8 * (kThreads / 32);
  static constexpr uint32_t kTmemCols = N == 64 ? 512 : 256;
  static constexpr uint32_t kTmemO = 2 * kTile;
  // the S product's A operand spans 64 rows from every chunk of Q: inside the allocation
  static_assert(kQ + kQBufs * kQBytes - N * 128 + 64 * 128 <= kBytes, "shared memory");
  static_assert(kBytes <= 227 * 1024, "shared memory");
  static_assert(kTmemO + kMTiles * N <= kTmemCols, "tensor memory");
};

struct LatentParams {
  void* out;
  float* lse;
  const int32_t* query_start_loc;  // null: uniform_q queries a sequence
  const int32_t* seq_lens;
  const int32_t* block_table;
  int64_t bt_stride, o_tok, o_head, lse_tok;
  int num_seqs, num_tokens, num_heads, uniform_q, max_query;
  int block_size, num_blocks, max_blocks;
  int group_heads, head_blocks, group_tokens;  // rows of a group = group_heads * group_tokens
  int teams, team_ctas;
  int64_t max_items;
  float scale_log2;
  float* part_o;    // [ctas][2][64][512]
  float* part_lse;  // [ctas][2][64], log2
  int4* desc;       // [ctas][2]: tiles before the share that ends an item (0: none), tiles a CTA; its rows
  unsigned int* err;
};

struct Seq {
  int q_begin, q_len, ctx, groups;
};

// One sequence's lengths; inconsistent metadata is reported and leaves it without groups.
__device__ __forceinline__ Seq sequence(const LatentParams& p, int b) {
  Seq s;
  if (p.query_start_loc != nullptr) {
    s.q_begin = p.query_start_loc[b];
    s.q_len = p.query_start_loc[b + 1] - s.q_begin;
  } else {
    s.q_begin = b * p.uniform_q;
    s.q_len = p.uniform_q;
  }
  if (s.q_begin < 0 || s.q_len < 0 || s.q_len > p.max_query || s.q_len > p.num_tokens - s.q_begin) {
    raise_device_error(p.err, NTB200_DEVERR_INDEX_RANGE);
    s.q_begin = s.q_len = 0;
  }
  s.ctx = p.seq_lens[b];
  if (s.ctx < 0) s.ctx = 0;
  if (int64_t(s.ctx) > int64_t(p.max_blocks) * p.block_size) {
    raise_device_error(p.err, NTB200_DEVERR_INDEX_RANGE);
    s.ctx = p.max_blocks * p.block_size;
  }
  s.groups = (s.q_len + p.group_tokens - 1) / p.group_tokens * p.head_blocks;
  return s;
}

// Keys that some row of group g sees, and its tiles (at least one: a group that sees nothing
// still has rows to write).
__device__ __forceinline__ int group_keys(const LatentParams& p, const Seq& s, int g) {
  const int last = min((g / p.head_blocks + 1) * p.group_tokens, s.q_len);
  return max(s.ctx - s.q_len + last, 0);
}
__device__ __forceinline__ int group_tiles(const LatentParams& p, const Seq& s, int g) {
  return max((group_keys(p, s, g) + kTile - 1) / kTile, 1);
}

// A CTA's share of one item: tiles [t0, t1) of n.
struct Piece {
  Seq s;
  int b, g, t0, t1, n, keys;
  __device__ __forceinline__ int valid(int t) const { return min(keys - t * kTile, kTile); }
};

// Walks a CTA's run of tiles; every role walks the same pieces.  `s` is sequence b.
struct Walk {
  Seq s;
  int b, g, t;
  int64_t left;
  __device__ __forceinline__ bool next(const LatentParams& p, int team, Piece& o) {
    while (left > 0) {
      if (g >= s.groups) {
        if (++b >= p.num_seqs) return false;
        s = sequence(p, b);
        g = team;
        t = 0;
        continue;
      }
      o.s = s;
      o.b = b;
      o.g = g;
      o.t0 = t;
      o.keys = group_keys(p, s, g);
      o.n = max((o.keys + kTile - 1) / kTile, 1);
      o.t1 = int64_t(o.n - t) < left ? o.n : t + int(left);
      left -= o.t1 - t;
      g += p.teams;
      t = 0;
      return true;
    }
    return false;
  }
};

// Tiles of sequence s that belong to this team.  With `skip` tiles to leave out: also the group
// and the tile in it that come next (when there are that many).
__device__ __forceinline__ int64_t team_tiles(const LatentParams& p, const Seq& s, int team, int64_t skip = -1,
                                              int* at_group = nullptr, int* at_tile = nullptr) {
  int64_t n = 0;
  if (p.teams > 1) {  // one group a sequence at most
    if (team >= s.groups) return 0;
    n = group_tiles(p, s, team);
    if (skip >= 0 && skip < n) *at_group = team, *at_tile = int(skip);
    return n;
  }
  int keys = s.ctx - s.q_len;
  for (int g = 0, last = 0; g < s.groups; g += p.head_blocks) {
    const int step = min(p.group_tokens, s.q_len - last);
    last += step;
    keys += step;
    const int tiles = max((keys + kTile - 1) / kTile, 1);
    const int64_t all = int64_t(tiles) * p.head_blocks;
    if (skip >= n && skip < n + all) {
      *at_group = g;
      int64_t rest = skip - n;
      for (; rest >= tiles; rest -= tiles) ++*at_group;
      *at_tile = int(rest);
      return n;
    }
    n += all;
  }
  return n;
}

__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, int group, int block, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %2, %2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(group), "r"(block), "r"(bar)
      : "memory");
}

// 16 TMEM lanes x 64 columns: registers 4 i + {0, 1} hold row lane / 4, columns 8 i + 2 (lane % 4)
// + {0, 1}; registers 4 i + {2, 3} the same columns of row lane / 4 + 8
__device__ __forceinline__ void tmem_ld_16x64(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// Barrier of the softmax warps that tells all of them whether any of them says yes.
__device__ __forceinline__ bool softmax_any(bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(v ? 1u : 0u), "n"(kSmThreads)
      : "memory");
  return r != 0;
}

// Operand tiles of the KV ring: 8-token groups kGroupBytes apart, a chunk's atom 1024 bytes.
__device__ __forceinline__ uint64_t ring_desc(uint32_t saddr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(1024 >> 4) << 16;         // next 64 columns (MN-major); unused K-major
  d |= static_cast<uint64_t>(kGroupBytes >> 4) << 32;  // next 8 tokens
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

// Writes this warp's 32 latent columns of every M tile: row c to dst + row_at[c] (none if
// negative), scaled by row_f[c].  Neighbouring lanes swap halves of two rows, so that a lane
// stores two adjacent columns of one row; 16 rows' loads, products and stores are in flight
// together.
template <typename T, typename O, int N>
__device__ __forceinline__ void write_rows(O* dst, uint32_t o_tmem, int quad, const float* row_f,
                                           const int64_t* row_at) {
  const int lane = threadIdx.x & 31;
  const int odd = lane & 1;
#pragma unroll 1
  for (int c0 = 0; c0 < N; c0 += 16) {
    float k[8];    // of the rows this lane stores: c0 + 2 i + odd
    int64_t at[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      k[i] = row_f[c0 + 2 * i + odd];
      at[i] = row_at[c0 + 2 * i + odd];
    }
#pragma unroll
    for (int j = 0; j < kMTiles; ++j) {
      const int col = j * 128 + quad * 32 + (lane & ~1);
      uint32_t v[16];
      __syncwarp();
      tmem_ld_16(o_tmem + j * N + c0, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t mine = odd ? v[2 * i + 1] : v[2 * i];
        const uint32_t other = __shfl_xor_sync(0xffffffffu, odd ? v[2 * i] : v[2 * i + 1], 1);
        float lo = __uint_as_float(odd ? other : mine) * k[i];
        float hi = __uint_as_float(odd ? mine : other) * k[i];
        if (k[i] == 0.f) lo = hi = 0.f;  // an empty row's O^T was never written
        if (at[i] >= 0) {
          if constexpr (sizeof(O) == 4) *reinterpret_cast<float2*>(dst + at[i] + col) = make_float2(lo, hi);
          else Pair<T>::store(dst + at[i] + col, lo, hi);
        }
      }
    }
  }
}

template <typename T, int N>
__global__ void __launch_bounds__(kThreads, 1)
    latent_attention_kernel(const __grid_constant__ CUtensorMap ql_map, const __grid_constant__ CUtensorMap qr_map,
                            const __grid_constant__ CUtensorMap c_map, const LatentParams p) {
  using L = Layout<N>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sm = smem_u32(smem);
  float* const row_f = reinterpret_cast<float*>(smem + L::kRowF);
  int64_t* const row_at = reinterpret_cast<int64_t*>(smem + L::kRowAt);
  uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + L::kBars);
  int* const start = reinterpret_cast<int*>(smem + L::kStart);  // b, g, t of the run's first tile, its sequence
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kStart + 28);
  int64_t* const scan = reinterpret_cast<int64_t*>(smem + L::kStart + 32);  // one a warp
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int team = blockIdx.x % p.teams;
  const int member = blockIdx.x / p.teams;
  pdl_trigger();
  pdl_wait();  // queries, cache and metadata come from the kernels before

  // ---- this CTA's run of its team's tiles ----
  if (threadIdx.x == 0) p.desc[int64_t(blockIdx.x) * 2] = make_int4(0, 0, 0, 0);  // ends no cut item yet
  Seq own;                    // this thread's first sequence
  int64_t own_tiles;
  int seqs = p.num_seqs;      // those that count
  for (;;) {
    own = {0, 0, 0, 0};
    int64_t mine = 0;
    int fall = seqs;
    if (int(threadIdx.x) < seqs) {
      own = sequence(p, threadIdx.x);
      mine = team_tiles(p, own, team);
    }
    own_tiles = mine;
    for (int b = threadIdx.x + kThreads; b < seqs; b += kThreads) mine += team_tiles(p, sequence(p, b), team);
    if (p.query_start_loc != nullptr)  // (compared once more here: as part of sequence() it cost 1.5 us of 99)
      for (int b = threadIdx.x; b < seqs; b += kThreads)
        if (p.query_start_loc[b + 1] < p.query_start_loc[b]) fall = min(fall, b);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if (lane == 0) scan[warp] = mine;
    if (!__syncthreads_or(fall < seqs)) break;
    // Start locations that fall: the sequences behind could own rows of those before, and two CTAs would
    // write them.  Those up to the first fall are counted again, the others left out.
    if (threadIdx.x == 0) start[0] = seqs;
    __syncthreads();
    atomicMin(&start[0], fall);
    __syncthreads();
    seqs = start[0];
  }
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) total += scan[w];
  const int64_t per = total <= 0x7fffffff - kMaxCtas ? int64_t((int(total) + p.team_ctas - 1) / p.team_ctas)
                                                     : (total + p.team_ctas - 1) / p.team_ctas;  // (slower)
  const int64_t begin = per * member;
  if (begin >= total) return;
  const int64_t count = min(per, total - begin);
  __syncthreads();
  int64_t carry = 0;
  for (int base = 0; base < seqs && carry <= begin; base += kThreads) {
    const int b = base + threadIdx.x;
    Seq sq = own;
    int64_t c = own_tiles;
    if (base > 0) {
      c = 0;
      if (b < seqs) {
        sq = sequence(p, b);
        c = team_tiles(p, sq, team);
      }
    }
    int64_t v = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += y;
    }
    if (lane == 31) scan[warp] = v;
    __syncthreads();
    int64_t before = carry, sum = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      before += w < warp ? scan[w] : 0;
      sum += scan[w];
    }
    const int64_t first = before + v - c;
    if (begin >= first && begin < first + c) {
      int g = 0, t = 0;
      team_tiles(p, sq, team, begin - first, &g, &t);
      start[0] = b, start[1] = g, start[2] = t;
      start[3] = sq.q_begin, start[4] = sq.q_len, start[5] = sq.ctx, start[6] = sq.groups;
    }
    carry += sum;
    __syncthreads();
  }

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kQBufs; ++i) mbar_init(&bars[L::kQFull + i], 1), mbar_init(&bars[L::kQEmpty + i], 1);
    for (int i = 0; i < kRing; ++i) mbar_init(&bars[L::kFull + i], 1), mbar_init(&bars[L::kEmpty + i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&bars[L::kSFull + i], 1), mbar_init(&bars[L::kSFree + i], kSmThreads / 32);
    mbar_init(&bars[L::kPFull], kSmThreads / 32);
    mbar_init(&bars[L::kPvDone], 1);
    mbar_init(&bars[L::kOFree], kSmThreads / 32);
    mbar_init(&bars[L::kMmaDone], 2);
    fence_mbar_init();
  }
  if (warp == 3) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(L::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  Walk walk = {{start[3], start[4], start[5], start[6]}, start[0], start[1], start[2], count};
  Piece pc;

  if (warp == 0) {
    // ------------------------------ TMA producer ------------------------------
    const uint32_t elected = elect_one();
    if (elected) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&ql_map)) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&qr_map)) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&c_map)) : "memory");
    }
    __syncwarp();
    const int rows = p.group_heads * p.group_tokens;
    uint32_t nq = 0, nu = 0;  // query loads and ring units so far
    bool ok = true;
    while (ok && walk.next(p, team, pc)) {
      const int32_t* const bt = p.block_table + int64_t(pc.b) * p.bt_stride;
      const int first = pc.t0 * kTileUnits;
      const int last = (min(pc.keys, pc.t1 * kTile) + kUnit - 1) / kUnit;  // units [first, last) hold keys
      // 32 units' page ids and groups at a time, one a lane, the next 32 fetched ahead
      int page = -1, group = 0, next_page = -1, next_group = 0;
      auto fetch = [&](int base) {
        const int tok = (base + lane) * kUnit;
        const int lb = tok / p.block_size;
        next_group = (tok - lb * p.block_size) / 8;
        next_page = base + lane < last ? __ldg(bt + lb) : 0;
      };
      fetch(first);
      const int qb = nq % L::kQBufs;
      uint64_t* const q_full = &bars[L::kQFull + qb];
      if (nq >= L::kQBufs && !mbar_spin_warp(&bars[L::kQEmpty + qb], (nq / L::kQBufs - 1) & 1, p.err)) break;
      if (elected) {
        mbar_arrive_expect_tx(q_full, kChunks * rows * 128);
        const int head = pc.g % p.head_blocks * p.group_heads;
        const int tok = pc.s.q_begin + pc.g / p.head_blocks * p.group_tokens;
        const uint32_t qdst = sm + L::kQ + qb * L::kQBytes;
        for (int c = 0; c < kChunks - 1; ++c) tma_load_3d(qdst + c * N * 128, &ql_map, c * 64, head, tok, smem_u32(q_full));
        tma_load_3d(qdst + (kChunks - 1) * N * 128, &qr_map, 0, head, tok, smem_u32(q_full));
      }
      __syncwarp();
      ++nq;
      // a tile is always four units of the ring, those past the last key empty
      const int end = (last + kTileUnits - 1) / kTileUnits * kTileUnits;
      for (int u = first; ok && u < end; ++u, ++nu) {
        const int i = (u - first) & 31;
        if (i == 0) {
          page = next_page;
          group = next_group;
          if (page < 0 || page >= p.num_blocks) {
            raise_device_error(p.err, NTB200_DEVERR_INDEX_RANGE);
            page = -1;  // outside the map: the rows read as zeros
          }
          if (u + 32 < last) fetch(u + 32);
        }
        const int at_page = __shfl_sync(0xffffffffu, page, i);
        const int at_group = __shfl_sync(0xffffffffu, group, i);
        const uint32_t s = nu % kRing;
        if (nu >= kRing && !mbar_spin_warp(&bars[L::kEmpty + s], (nu / kRing - 1) & 1, p.err)) {
          ok = false;
          break;
        }
        if (elected) {
          if (u < last) {
            mbar_arrive_expect_tx(&bars[L::kFull + s], kUnitBytes);
            tma_load_5d(sm + L::kKv + s * kUnitBytes, &c_map, at_group, at_page, smem_u32(&bars[L::kFull + s]));
          } else {
            mbar_arrive(&bars[L::kFull + s]);
          }
        }
        __syncwarp();
      }
    }
    // drain the copies that may still be in flight
    for (uint32_t i = nq > L::kQBufs ? nq - L::kQBufs : 0; i < nq; ++i)
      mbar_spin_warp(&bars[L::kQFull + i % L::kQBufs], (i / L::kQBufs) & 1, p.err);
    for (uint32_t i = nu > kRing ? nu - kRing : 0; i < nu; ++i)
      mbar_spin_warp(&bars[L::kFull + i % kRing], (i / kRing) & 1, p.err);
  } else if (warp == 1) {
    // -------------------------- MMA issuer: S = Q C^T --------------------------
    const uint32_t elected = elect_one();
    const uint32_t idesc = make_idesc(std::is_same<T, __nv_bfloat16>::value, 64, kTile);
    uint32_t nq = 0, nu = 0, g = 0;
    bool ok = true;
    while (ok && walk.next(p, team, pc)) {
      const int qb = nq % L::kQBufs;
      if (!mbar_spin_warp(&bars[L::kQFull + qb], (nq / L::kQBufs) & 1, p.err)) break;
      const uint64_t a0 = sw128_kmajor_desc(sm + L::kQ + qb * L::kQBytes);
      for (int t = pc.t0; t < pc.t1; ++t, ++g) {
        const int s = g & 1;
        // the softmax has read this buffer's scores of two tiles ago
        if (g >= 2) ok = mbar_spin_warp(&bars[L::kSFree + s], (g / 2 - 1) & 1, p.err);
        if (pc.valid(t) > 0) {
          for (int i = 0; i < kTileUnits && ok; ++i)
            ok = mbar_spin_warp(&bars[L::kFull + (nu + i) % kRing], ((nu + i) / kRing) & 1, p.err);
          if (!ok) break;
          tc_fence_after();
          const uint64_t b0 = ring_desc(sm + L::kKv + nu % kRing * kUnitBytes);
#pragma unroll
          for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_elected(tmem + s * kTile, a0 + c * (N * 128 >> 4) + 2 * k, b0 + c * (1024 >> 4) + 2 * k, idesc,
                           (c | k) ? 1u : 0u, elected);
          nu += kTileUnits;
        }
        if (!ok) break;
        commit_elected(&bars[L::kSFull + s], elected);
      }
      commit_elected(&bars[L::kQEmpty + qb], elected);
      ++nq;
    }
    // every issued MMA completes before TMEM may be released
    commit_elected(&bars[L::kMmaDone], elected);
    mbar_spin_warp(&bars[L::kMmaDone], 0, p.err);
  } else if (warp == 2) {
    // ------------------------ MMA issuer: O^T += C^T P^T ------------------------
    const uint32_t elected = elect_one();
    const uint32_t idesc = make_idesc(std::is_same<T, __nv_bfloat16>::value, 128, N) | (1u << 15);  // A MN-major
    const uint64_t b0 = sw128_kmajor_desc(sm + L::kP);
    uint32_t nu = 0, g = 0, pieces = 0;
    bool ok = true;
    while (ok && walk.next(p, team, pc)) {
      for (int t = pc.t0; t < pc.t1; ++t, ++g) {
        // the first product of a piece overwrites O^T: the one before has been written out
        ok = mbar_spin_warp(&bars[L::kPFull], g & 1, p.err) &&
             (t > pc.t0 || pieces == 0 || mbar_spin_warp(&bars[L::kOFree], (pieces - 1) & 1, p.err));
        if (!ok) break;
        const int valid = pc.valid(t);
        if (valid > 0) {
          tc_fence_after();
          const int steps = (valid + kUnit - 1) / kUnit;
          const uint64_t a0 = ring_desc(sm + L::kKv + nu % kRing * kUnitBytes);
#pragma unroll
          for (int k = 0; k < kTileUnits; ++k) {
            if (k < steps) {
#pragma unroll
              for (int j = 0; j < kMTiles; ++j)
                umma_elected(tmem + L::kTmemO + j * N, a0 + k * (kUnitBytes >> 4) + j * (2048 >> 4), b0 + 2 * k, idesc,
                             (t > pc.t0 || k > 0) ? 1u : 0u, elected);
            }
            commit_elected(&bars[L::kEmpty + (nu + k) % kRing], elected);
          }
          nu += kTileUnits;
        }
        commit_elected(&bars[L::kPvDone], elected);
      }
      ++pieces;
    }
    commit_elected(&bars[L::kMmaDone], elected);
    mbar_spin_warp(&bars[L::kMmaDone], 0, p.err);
  } else if (warp >= kFirstSmWarp) {
    // ------------------------------ softmax + output ------------------------------
    // The M = 64 product leaves row r in TMEM lane 32 (r / 16) + r % 16: warp `quad` has rows
    // 16 quad .. + 16, this lane the columns 8 i + 2 (lane % 4) + {0, 1} of rows r0 and r0 + 8.  O^T
    // covers all lanes: every warp rescales and writes its 32 latent columns of each M tile.
    // A wait that gave up is told to the other warps at the next barrier, where all leave.
    const int quad = warp & 3;
    const bool active = quad * 16 < N;
    const int r0 = quad * 16 + (lane >> 2);
    const uint32_t lanes = uint32_t(quad * 32) << 16;
    const uint32_t o_tmem = tmem + L::kTmemO + lanes;
    const int col0 = 2 * (lane & 3);
    uint32_t g = 0, nu = 0, pieces = 0;
    bool bad = false;
    while (!bad && walk.next(p, team, pc)) {
      const int tok0 = pc.g / p.head_blocks * p.group_tokens;
      const int head0 = pc.g % p.head_blocks * p.group_heads;
      // rows of the group: (token, head) = (row / group_heads, row % group_heads); this lane's two
      int tok[2], head[2], limit[2];
      bool there[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = r0 + 8 * i;
        const int rt = row / p.group_heads;
        tok[i] = tok0 + rt;
        head[i] = head0 + row - rt * p.group_heads;
        there[i] = active && rt < p.group_tokens && tok[i] < pc.s.q_len && head[i] < p.num_heads;
        limit[i] = there[i] ? max(pc.s.ctx - pc.s.q_len + tok[i] + 1, 0) : 0;  // sees keys [0, limit)
      }
      // a cut item's share: the CTA's last piece begins it (t0 = 0), its first one continues it
      const bool whole = pc.t0 == 0 && pc.t1 == pc.n;
      const int64_t share = int64_t(blockIdx.x) * 2 + (pc.t0 == 0 ? 1 : 0);
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
      bool left = false;
      for (int t = pc.t0; t < pc.t1; ++t, ++g) {
        const int s = g & 1;
        const int valid = pc.valid(t);
        bad = bad || !mbar_spin_warp(&bars[L::kSFull + s], (g / 2) & 1, p.err);
        tc_fence_after();
        float x[32];
        float alpha[2] = {1.f, 1.f};
        bool grow = false;
        if (active) {
          {
            uint32_t v[32];
            __syncwarp();
            tmem_ld_16x64(tmem + lanes + s * kTile, v);
#pragma unroll
            for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(v[i]);
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int seen = limit[h] - t * kTile - col0;
            if (seen < kTile - col0) {
#pragma unroll
              for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  if (8 * i + e >= seen) x[4 * i + 2 * h + e] = -INFINITY;
            }
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 8; ++i) mx = fmaxf(mx, fmaxf(x[4 * i + 2 * h], x[4 * i + 2 * h + 1]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float m_new = fmaxf(m[h], mx * p.scale_log2);  // the scale is positive
            if (m_new > m[h] + kRescaleLog2) {  // also true for the first finite maximum
              alpha[h] = hw_exp2(m[h] - m_new);
              m[h] = m_new;
              l[h] *= alpha[h];
              grow = true;
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[L::kSFree + s]);
        const bool news = softmax_any(grow || bad);
        if (t == pc.t0 && active && (lane & 3) == 0) {  // (every warp has written the piece before out)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            row_at[r0 + 8 * h] = !there[h] ? -1
                                 : whole   ? int64_t(pc.s.q_begin + tok[h]) * p.o_tok + int64_t(head[h]) * p.o_head
                                           : (share * kMaxRows + r0 + 8 * h) * kLatent;
        }
        if (news) {
          if ((lane & 3) == 0 && active) row_f[r0] = alpha[0], row_f[r0 + 8] = alpha[1];
          left = softmax_any(bad);
          if (left) break;
        }
        uint32_t pk[16];
        if (active) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float m_use = m[h] == -INFINITY ? 0.f : m[h] - kBias<T>;
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float p0 = hw_exp2(fmaf(x[4 * i + 2 * h], p.scale_log2, -m_use));
              const float p1 = hw_exp2(fmaf(x[4 * i + 2 * h + 1], p.scale_log2, -m_use));
              sum += p0 + p1;
              Pair<T>::store(reinterpret_cast<T*>(&pk[2 * i + h]), p0, p1);
            }
            l[h] += sum;
          }
        }
        // P and O^T are free once the product of the tile before is complete
        if (g >= 1) bad = bad || !mbar_spin_warp(&bars[L::kPvDone], (g - 1) & 1, p.err);
        if (news && t > pc.t0) {
          tc_fence_after();
#pragma unroll 1
          for (int j = 0; j < kMTiles; ++j)
#pragma unroll 1
            for (int c0 = 0; c0 < N; c0 += 16) {
              uint32_t v[16];
              __syncwarp();
              tmem_ld_16(o_tmem + j * N + c0, v);
#pragma unroll
              for (int c = 0; c < 16; ++c) v[c] = __float_as_uint(__uint_as_float(v[c]) * row_f[c0 + c]);
              tmem_st_16(o_tmem + j * N + c0, v);
            }
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        }
        if (active) {
          // P [row, token], 128-byte swizzled rows: 8 tokens a 16-byte unit, two a lane
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int row = r0 + 8 * h;
            uint8_t* const prow = smem + L::kP + row * 128 + (lane & 3) * 4;
#pragma unroll
            for (int i = 0; i < 8; ++i) *reinterpret_cast<uint32_t*>(prow + ((i ^ (row & 7)) << 4)) = pk[2 * i + h];
          }
        }
        if (valid > 0) {
          if (valid & 15) {
            // rows past the last visible key, up to the product's next step of 16, hold whatever
            // memory held there: zeroed, so that P = 0 never meets a non-finite value
            const int n = 16 - (valid & 15);
            uint8_t* const tile = smem + L::kKv + nu % kRing * kUnitBytes;
            for (int i = threadIdx.x - 32 * kFirstSmWarp; i < n * 64; i += kSmThreads) {
              const int row = valid + (i >> 6);
              *reinterpret_cast<uint4*>(tile + (row >> 3) * kGroupBytes + ((i >> 3) & 7) * 1024 + (row & 7) * 128 +
                                        (i & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
          }
          nu += kTileUnits;
        }
        fence_proxy_async_smem();  // P and the zeros -> tensor core
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[L::kPFull]);
      }
      if (left) break;
      // O^T is final once the piece's last product is complete
      bad = bad || !mbar_spin_warp(&bars[L::kPvDone], (g - 1) & 1, p.err);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = r0 + 8 * h;
        float sum = l[h];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if (active && (lane & 3) == 0) {
          const float lse2 = sum == 0.f ? -INFINITY : m[h] - kBias<T> + log2f(sum);
          row_f[row] = sum == 0.f ? 0.f : 1.f / sum;
          if (!there[h]) continue;
          if (!whole) p.part_lse[share * kMaxRows + row] = lse2;
          else if (p.lse != nullptr) p.lse[int64_t(pc.s.q_begin + tok[h]) * p.lse_tok + head[h]] = lse2 * 0.6931471805599453f;
        }
      }
      if (pc.t0 > 0 && pc.t1 == pc.n && warp == kFirstSmWarp && lane == 0) {  // this CTA ends a cut item
        p.desc[int64_t(blockIdx.x) * 2] = make_int4(pc.t0, int(min(per, int64_t(0x7fffffff))), 0, 0);
        p.desc[int64_t(blockIdx.x) * 2 + 1] = make_int4(pc.s.q_begin + tok0, pc.s.q_len - tok0, head0, 0);
      }
      if (softmax_any(bad)) break;
      tc_fence_after();
      if (whole) write_rows<T, T, N>(static_cast<T*>(p.out), o_tmem, quad, row_f, row_at);
      else write_rows<T, float, N>(p.part_o, o_tmem, quad, row_f, row_at);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[L::kOFree]);  // the next piece may overwrite O^T
      ++pieces;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 3) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::kTmemCols) : "memory");
  }
}

// Joins the shares of every item that was cut; block x takes the x-th CTA whose first piece ends
// one.  Every CTA between the item's first (whose last piece begins it) and that one had nothing
// else to do, so their number follows from the tiles before and the tiles a CTA.  128 threads sum
// four columns each of a row.  PARTS = 4: a block's four sets of 128 share one row, each with every
// fourth share (few items, so many shares each: 32 shares of 16 rows took 10 us on two SMs);
// PARTS = 1: they take four rows, twice (many items, a few shares each).
constexpr int kJoinSets = 4;
constexpr int join_rows(int parts) { return parts == 1 ? 2 * kJoinSets : 1; }

template <typename T, int PARTS>
__global__ void __launch_bounds__(kJoinSets * 128) latent_join_kernel(const LatentParams p) {
  __shared__ float weight[kJoinSets][kMaxCtas];
  __shared__ float tops[kJoinSets][4];
  __shared__ float4 sums[PARTS == 1 ? 1 : kJoinSets][128];
  __shared__ int ends[kJoinSets * 4], found;
  const int set = threadIdx.x >> 7, col = threadIdx.x & 127;
  pdl_trigger();
  pdl_wait();
  // ---- the x-th CTA that ends a cut item ----
  const int ctas = p.teams * p.team_ctas;
  const bool mine = threadIdx.x < ctas && p.desc[2 * threadIdx.x].x != 0;
  const unsigned votes = __ballot_sync(0xffffffffu, mine);
  if ((threadIdx.x & 31) == 0) ends[threadIdx.x >> 5] = __popc(votes);
  if (threadIdx.x == 0) found = -1;
  __syncthreads();
  int before = __popc(votes & ((1u << (threadIdx.x & 31)) - 1));
  for (int w = 0; w < (threadIdx.x >> 5); ++w) before += ends[w];
  if (mine && before == blockIdx.x) found = threadIdx.x;
  __syncthreads();
  const int cta = found;
  if (cta < 0) return;
  const int4 end = p.desc[2 * cta];
  const int4 where = p.desc[2 * cta + 1];
  const int n = 1 + (end.x + end.y - 1) / end.y;
  const int first = cta - (n - 1) * p.teams;
  auto share = [&](int i) { return int64_t(i == 0 ? first * 2 + 1 : (first + i * p.teams) * 2); };
#pragma unroll 1
  for (int k = 0; k < (PARTS == 1 ? 2 : 1); ++k) {
    const int r = blockIdx.y * join_rows(PARTS) + (PARTS == 1 ? k * kJoinSets + set : 0);
    const int tok = r / p.group_heads;
    const int head = where.z + r - tok * p.group_heads;
    const bool there = tok < p.group_tokens && tok < where.y && head < p.num_heads;
    float top = -INFINITY;
    for (int i = col; there && i < n; i += 128) {
      const float l = p.part_lse[share(i) * kMaxRows + r];
      weight[set][i] = l;
      top = fmaxf(top, l);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((col & 31) == 0) tops[set][col >> 5] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[set][0], tops[set][1]), fmaxf(tops[set][2], tops[set][3]));
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (there) {
      for (int i = col; i < n; i += 128) weight[set][i] = exp2f(weight[set][i] - ref);
    }
    __syncthreads();
    if (there) {
#pragma unroll 8
      for (int i = PARTS == 1 ? 0 : set; i < n; i += PARTS) {
        const float w = weight[set][i];
        const float4 o = reinterpret_cast<const float4*>(p.part_o + (share(i) * kMaxRows + r) * kLatent)[col];
        sum += w;
        acc.x += w * o.x, acc.y += w * o.y, acc.z += w * o.z, acc.w += w * o.w;
      }
    }
    if constexpr (PARTS > 1) {
      sums[set][col] = acc;
      if (col == 0) tops[set][0] = sum;
      __syncthreads();
      if (set > 0) return;
#pragma unroll
      for (int q = 1; q < PARTS; ++q) {
        const float4 o = sums[q][col];
        sum += tops[q][0];
        acc.x += o.x, acc.y += o.y, acc.z += o.z, acc.w += o.w;
      }
    }
    if (there) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const float y[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
      T* const o = static_cast<T*>(p.out) + int64_t(where.x + tok) * p.o_tok + int64_t(head) * p.o_head;
      *reinterpret_cast<Vec<T, 4>*>(o + col * 4) = pack_f<T, 4>(y);
      if (p.lse != nullptr && col == 0)
        p.lse[int64_t(where.x + tok) * p.lse_tok + head] = sum == 0.f ? -INFINITY : (ref + log2f(sum)) * 0.6931471805599453f;
    }
    if constexpr (PARTS == 1) __syncthreads();
  }
}

// [tokens, heads, dim] queries: box = group_tokens x group_heads x 64 columns
int make_query_map(CUtensorMap* map, const void* base, bool bf16, int64_t dim, int64_t tokens, int64_t heads,
                   int64_t tok_stride, int64_t head_stride, int group_tokens, int group_heads) {
  EncodeTiledFn enc = encode_fn();
  if (enc == nullptr) return fail(NTB200_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const cuuint64_t dims[3] = {cuuint64_t(dim), cuuint64_t(heads), cuuint64_t(tokens)};
  const cuuint64_t strides[2] = {cuuint64_t((heads > 1 ? head_stride : dim) * 2),
                                 cuuint64_t((tokens > 1 ? tok_stride : dim) * 2)};
  const cuuint32_t box[3] = {64, cuuint32_t(group_heads), cuuint32_t(group_tokens)};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                         const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(NTB200_ERR_CUDA, "cuTensorMapEncodeTiled (latent q) failed (%d)", int(r));
  return NTB200_OK;
}

// the cache [blocks, block_size, 576] as (64 columns, 8 tokens, 9 chunks, groups of 8 tokens,
// blocks): box = 16 tokens' whole rows, laid down group by group, chunk by chunk
int make_cache_map(CUtensorMap* map, const void* base, bool bf16, int64_t blocks, int64_t block_size,
                   int64_t block_stride, int64_t page_stride) {
  EncodeTiledFn enc = encode_fn();
  if (enc == nullptr) return fail(NTB200_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const cuuint64_t dims[5] = {64, 8, cuuint64_t(kChunks), cuuint64_t(block_size / 8), cuuint64_t(blocks)};
  const cuuint64_t strides[4] = {cuuint64_t(page_stride * 2), 128, cuuint64_t(page_stride * 16),
                                 cuuint64_t((blocks > 1 ? block_stride : block_size * page_stride) * 2)};
  const cuuint32_t box[5] = {64, 8, cuuint32_t(kChunks), kUnit / 8, 1};
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  const CUresult r = enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5,
                         const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(NTB200_ERR_CUDA, "cuTensorMapEncodeTiled (latent cache) failed (%d)", int(r));
  return NTB200_OK;
}

template <typename T, int N>
int launch_latent(const CUtensorMap& ql, const CUtensorMap& qr, const CUtensorMap& c, const LatentParams& p, int slot,
                  cudaStream_t s) {
  int st = ensure_smem_attribute(reinterpret_cast<const void*>(latent_attention_kernel<T, N>), Layout<N>::kBytes, slot);
  if (st != NTB200_OK) return st;
  const unsigned ctas = unsigned(p.teams * p.team_ctas);
  st = launch_kernel("latent_attention", latent_attention_kernel<T, N>, dim3(ctas), dim3(kThreads), Layout<N>::kBytes,
                     s, ql, qr, c, p);
  if (st != NTB200_OK || p.team_ctas == 1) return st;  // one CTA a team cuts no item
  // blocks for as many items as can be cut; one row each where an item has over three shares on average
  const unsigned rows = unsigned(p.group_heads * p.group_tokens);
  const unsigned items = unsigned(std::min<int64_t>(p.max_items, ctas));
  if (ctas > 3 * items)
    return launch_kernel("latent_attention (join)", latent_join_kernel<T, 4>, dim3(items, rows), dim3(kJoinSets * 128), 0, s, p);
  return launch_kernel("latent_attention (join)", latent_join_kernel<T, 1>,
                       dim3(items, unsigned(ceil_div(rows, join_rows(1)))), dim3(kJoinSets * 128), 0, s, p);
}

template <typename T>
int by_rows(const CUtensorMap& ql, const CUtensorMap& qr, const CUtensorMap& c, const LatentParams& p, int slot,
            cudaStream_t s) {
  const int rows = p.group_heads * p.group_tokens;
  if (rows <= 16) return launch_latent<T, 16>(ql, qr, c, p, slot, s);
  if (rows <= 32) return launch_latent<T, 32>(ql, qr, c, p, slot + 1, s);
  return launch_latent<T, 64>(ql, qr, c, p, slot + 2, s);
}

constexpr int64_t kShareFloats = int64_t(kMaxRows) * kLatent;
// per CTA: two shares of 64 x 512, their 64 log-sums, and their descriptors
constexpr int64_t kBytesPerCta = 2 * (kShareFloats * 4 + kMaxRows * 4 + 32);

}  // namespace
}  // namespace ntb200

extern "C" size_t ntb200_latent_attention_workspace_size(void) {
  return size_t(ntb200::num_sms()) * size_t(ntb200::kBytesPerCta);
}

extern "C" int ntb200_latent_attention(
    void* out, float* lse, const void* q_latent, const void* q_rope, const void* kv_cache,
    const int32_t* query_start_loc, const int32_t* seq_lens, const int32_t* block_tables, int64_t num_seqs,
    int64_t num_tokens, int64_t num_heads, int64_t latent_dim, int64_t rope_dim, int64_t block_size,
    int64_t num_blocks, int64_t max_blocks_per_seq, int64_t block_table_stride, int64_t max_query_len,
    int64_t max_seq_len, float scale, int64_t ql_token_stride, int64_t ql_head_stride, int64_t qr_token_stride,
    int64_t qr_head_stride, int64_t out_token_stride, int64_t out_head_stride, int64_t lse_token_stride,
    int64_t cache_block_stride, int64_t cache_page_stride, void* workspace, size_t workspace_bytes, int dtype,
    void* stream) {
  using namespace ntb200;
  if (dtype != NTB200_DTYPE_BF16 && dtype != NTB200_DTYPE_F16)
    return fail(NTB200_ERR_UNSUPPORTED_DTYPE, "latent_attention: dtype %d (bf16/f16 only)", dtype);
  if (latent_dim != kLatent || rope_dim != kRope || block_size <= 0 || block_size % 16 != 0)
    return fail(NTB200_ERR_UNSUPPORTED_SHAPE,
                "latent_attention: latent_dim %lld / rope_dim %lld / block_size %lld (512 / 64 / a multiple of 16)",
                (long long)latent_dim, (long long)rope_dim, (long long)block_size);
  if (num_seqs < 0 || num_tokens < 0 || num_heads <= 0 || num_blocks < 0 || max_blocks_per_seq < 0 ||
      block_table_stride < max_blocks_per_seq || max_query_len < 0)
    return fail(NTB200_ERR_INVALID_ARGUMENT, "latent_attention: bad sizes");
  if (!(scale > 0.f)) return fail(NTB200_ERR_INVALID_ARGUMENT, "latent_attention: scale must be positive");
  if (query_start_loc == nullptr && num_seqs > 0 && num_tokens % num_seqs != 0)
    return fail(NTB200_ERR_INVALID_ARGUMENT, "latent_attention: without query_start_loc every sequence has num_tokens / num_seqs queries");
  if (num_seqs == 0 || num_tokens == 0 || (query_start_loc != nullptr && max_query_len == 0)) return NTB200_OK;
  if (num_seqs > 0x7fffffff || num_tokens > 0x7fffffff || num_heads > 65535 || num_blocks > 0x7fffffff ||
      max_blocks_per_seq > (0x7fffffff - 1024) / block_size)
    return fail(NTB200_ERR_UNSUPPORTED_SHAPE, "latent_attention: sizes beyond the launch limits");
  if (!out || !q_latent || !q_rope || !seq_lens || (max_blocks_per_seq > 0 && (!block_tables || !kv_cache || num_blocks == 0)))
    return fail(NTB200_ERR_INVALID_ARGUMENT, "latent_attention: null pointer");
  if (!aligned16(out) || !aligned16(q_latent) || !aligned16(q_rope) || !aligned16(kv_cache) || ql_token_stride % 8 ||
      ql_head_stride % 8 || qr_token_stride % 8 || qr_head_stride % 8 || out_token_stride % 8 || out_head_stride % 8 ||
      cache_block_stride % 8 || cache_page_stride % 8)
    return fail(NTB200_ERR_MISALIGNED, "latent_attention: pointers 16-byte aligned, strides multiples of 8");
  if (max_blocks_per_seq > 0 && cache_page_stride < kLatent + kRope)
    return fail(NTB200_ERR_INVALID_ARGUMENT, "latent_attention: cache token stride below its row");
  const int64_t sms = num_sms() < kMaxCtas ? num_sms() : kMaxCtas;
  if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0 ||
      workspace_bytes < ntb200_latent_attention_workspace_size())
    return fail(NTB200_ERR_WORKSPACE, "latent_attention: workspace of %zu bytes, 256-byte aligned",
                ntb200_latent_attention_workspace_size());
  const bool bf16 = dtype == NTB200_DTYPE_BF16;
  LatentParams p = {};
  p.out = out;
  p.lse = lse;
  p.query_start_loc = query_start_loc;
  p.seq_lens = seq_lens;
  p.block_table = block_tables;
  p.bt_stride = block_table_stride;
  p.o_tok = out_token_stride;
  p.o_head = out_head_stride;
  p.lse_tok = lse_token_stride;
  p.num_seqs = int(num_seqs);
  p.num_tokens = int(num_tokens);
  p.num_heads = int(num_heads);
  p.uniform_q = query_start_loc == nullptr ? int(num_tokens / num_seqs) : 0;
  p.max_query = query_start_loc == nullptr ? p.uniform_q : int(std::min<int64_t>(max_query_len, num_tokens));
  p.block_size = int(block_size);
  p.num_blocks = int(num_blocks);
  p.max_blocks = int(max_blocks_per_seq);
  p.head_blocks = int(ceil_div(num_heads, kMaxRows));
  p.group_heads = int(ceil_div(num_heads, p.head_blocks));
  p.group_tokens = std::min(kMaxRows / p.group_heads, p.max_query);
  p.scale_log2 = scale * 1.4426950408889634f;  // softmax in the exp2 domain
  p.err = device_error_word();
  const int64_t groups = ceil_div(p.max_query, p.group_tokens) * p.head_blocks;
  p.teams = groups <= kMaxTeams ? int(groups) : 1;
  p.max_items = groups * num_seqs;
  const int64_t cap = max_blocks_per_seq * block_size;
  const int64_t keys = max_seq_len > 0 && max_seq_len < cap ? max_seq_len : cap;
  // no more CTAs than the batch can have tiles
  const int64_t tiles = std::max<int64_t>(ceil_div(keys, kTile), 1) * ceil_div(groups, p.teams);
  const int64_t most = std::max<int64_t>(sms / p.teams, 1);
  p.team_ctas = int(tiles >= most || num_seqs >= most ? most : std::min(most, tiles * num_seqs));
  const int64_t ctas = int64_t(p.teams) * p.team_ctas;
  p.part_o = static_cast<float*>(workspace);
  p.part_lse = p.part_o + ctas * 2 * kShareFloats;
  p.desc = reinterpret_cast<int4*>(p.part_lse + ctas * 2 * kMaxRows);
  CUtensorMap ql, qr, c;
  int st = make_query_map(&ql, q_latent, bf16, kLatent, num_tokens, num_heads, ql_token_stride, ql_head_stride,
                          p.group_tokens, p.group_heads);
  if (st != NTB200_OK) return st;
  st = make_query_map(&qr, q_rope, bf16, kRope, num_tokens, num_heads, qr_token_stride, qr_head_stride, p.group_tokens,
                      p.group_heads);
  if (st != NTB200_OK) return st;
  if (max_blocks_per_seq > 0) {
    st = make_cache_map(&c, kv_cache, bf16, num_blocks, block_size, cache_block_stride, cache_page_stride);
    if (st != NTB200_OK) return st;
  } else {
    c = ql;  // never read: every context is empty
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return bf16 ? by_rows<__nv_bfloat16>(ql, qr, c, p, 128, s) : by_rows<__half>(ql, qr, c, p, 131, s);
}
