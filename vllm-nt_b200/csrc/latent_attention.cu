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
// One tile, 640 threads:
//   warp 0      TMA: the item's queries (9 chunks of 64 columns), then per tile the rotary
//               chunk and 4 pairs of latent chunks into two rings, page by page.
//   warp 1      S = Q C^T on tcgen05 (M = 128: rows past the group's are whatever shared memory
//               holds, and their lanes are never read; N = 64 tokens), two S buffers.
//   warp 2      O^T += C^T P^T: the cached rows as the MN-major A operand (M = 128 latent
//               columns, four times), P [rows, tokens] as B.  O^T takes 4 x rows TMEM columns
//               where O would need all 512, which leaves room for S and lets the tile that S
//               was made from be used as it lies.
//   warps 4-19  softmax (a lane a query row, 16 of the tile's tokens a warp), the running max
//               refreshed only when it grows by over 2^8 (O^T is rescaled then), the output.
//
// Bound: HBM while 2 * rows * 1088 operations a token take less time than its 1152 bytes.
#include <algorithm>

#include "common.cuh"
#include "tcgen05.cuh"

namespace ntb200 {
namespace {

constexpr int kLatent = 512;
constexpr int kRope = 64;
constexpr int kChunks = (kLatent + kRope) / 64;  // 64-column chunks of a row; the last is rotary
constexpr int kTile = 64;                        // cached tokens a tile
constexpr int kChunkBytes = kTile * 128;         // 64 tokens x 64 columns
constexpr int kPairBytes = 2 * kChunkBytes;
constexpr int kPairs = kLatent / 128;
constexpr int kMaxRows = 64;                     // query rows a group
constexpr int kSmWarps = 16;
constexpr int kFirstSmWarp = 4;
constexpr int kThreads = 32 * (kFirstSmWarp + kSmWarps);
constexpr int kParts = 4;                        // warps that share a row's 64 tokens
constexpr int kPartCols = kTile / kParts;
constexpr int kMaxTeams = 8;
constexpr float kRescaleLog2 = 8.0f;

template <int N>
struct Layout {
  static constexpr int kQBufs = N == 64 ? 1 : 2;
  static constexpr int kRopeSlots = 2;
  static constexpr int kPairSlots = N == 16 ? 10 : 8;
  static constexpr int kQBytes = kChunks * N * 128;
  static constexpr int kQ = 0;
  static constexpr int kRopeRing = kQ + kQBufs * kQBytes;
  static constexpr int kPairRing = kRopeRing + kRopeSlots * kChunkBytes;
  static constexpr int kP = kPairRing + kPairSlots * kPairBytes;
  static constexpr int kRed = kP + N * 128;                       // [2][kParts][64] floats
  static constexpr int kBars = kRed + 2 * kParts * kMaxRows * 4;  // mbarriers
  static constexpr int kQFull = 0, kQEmpty = kQFull + kQBufs, kRopeFull = kQEmpty + kQBufs,
                       kRopeEmpty = kRopeFull + kRopeSlots, kPairFull = kRopeEmpty + kRopeSlots,
                       kPairEmpty = kPairFull + kPairSlots, kSFull = kPairEmpty + kPairSlots, kSFree = kSFull + 2,
                       kPFull = kSFree + 2, kPvDone = kPFull + 1, kOFree = kPvDone + 1, kMmaDone = kOFree + 1,
                       kExch = kMmaDone + 1, kNumBars = kExch + 1;
  static constexpr int kStart = kBars + 8 * kNumBars;  // the run's first tile, TMEM base, scan scratch
  static constexpr int kBytes = kStart + 64 + 8 * (kThreads / 32);
  static constexpr uint32_t kTmemCols = N == 64 ? 512 : 256;
  static constexpr uint32_t kTmemO = 2 * kTile;
  // the S product's A operand spans 128 rows from every chunk of Q: inside the allocation
  static_assert(kQ + kQBufs * kQBytes - N * 128 + 128 * 128 <= kBytes, "shared memory");
  static_assert(kBytes <= 227 * 1024, "shared memory");
  static_assert(kTmemO + kPairs * N <= kTmemCols, "tensor memory");
};

struct LatentParams {
  void* out;
  float* lse;
  const int32_t* query_start_loc;  // null: uniform_q queries a sequence
  const int32_t* seq_lens;
  const int32_t* block_table;
  int64_t bt_stride, o_tok, o_head, lse_tok;
  int num_seqs, num_tokens, num_heads, uniform_q, max_query;
  int block_size, sub_rows, num_blocks, max_blocks;
  int group_heads, head_blocks, group_tokens;  // rows of a group = group_heads * group_tokens
  int teams, team_ctas;
  float scale_log2;
  float* part_o;    // [ctas][2][64][512]
  float* part_lse;  // [ctas][2][64], log2
  int4* desc;       // [ctas][2][2]
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

// Walks a CTA's run of tiles; every role walks the same pieces.
struct Walk {
  int b, g, t;
  int64_t left;
  __device__ __forceinline__ bool next(const LatentParams& p, int team, Piece& o) {
    while (left > 0 && b < p.num_seqs) {
      o.s = sequence(p, b);
      if (g >= o.s.groups) {
        ++b;
        g = team;
        t = 0;
        continue;
      }
      o.b = b;
      o.g = g;
      o.t0 = t;
      o.keys = group_keys(p, o.s, g);
      o.n = group_tiles(p, o.s, g);
      o.t1 = int64_t(o.n - t) < left ? o.n : t + int(left);
      left -= o.t1 - t;
      g += p.teams;
      t = 0;
      return true;
    }
    return false;
  }
};

// tiles of sequence b that belong to this team
__device__ __forceinline__ int64_t team_tiles(const LatentParams& p, int b, int team) {
  const Seq s = sequence(p, b);
  int64_t n = 0;
  for (int g = team; g < s.groups; g += p.teams) n += group_tiles(p, s, g);
  return n;
}

__device__ __forceinline__ float hw_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void tmem_st_16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// The running max m of a row is subtracted as m - kBias: fp16 weights then span 2^7 .. 2^15 at
// the row's largest score and reach 2^-31 of it before they vanish (bf16 has fp32's range).
template <typename T>
constexpr float kBias = 0.f;
template <>
constexpr float kBias<__half> = 7.f;

template <typename T, int N>
__global__ void __launch_bounds__(kThreads, 1)
    latent_attention_kernel(const __grid_constant__ CUtensorMap ql_map, const __grid_constant__ CUtensorMap qr_map,
                            const __grid_constant__ CUtensorMap c_map, const LatentParams p) {
  using L = Layout<N>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sm = smem_u32(smem);
  float* const red = reinterpret_cast<float*>(smem + L::kRed);
  uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + L::kBars);
  int* const start = reinterpret_cast<int*>(smem + L::kStart);  // b, g, t of the run's first tile
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kStart + 16);
  int64_t* const total_slot = reinterpret_cast<int64_t*>(smem + L::kStart + 32);
  int64_t* const scan = reinterpret_cast<int64_t*>(smem + L::kStart + 64);  // one a warp
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int team = blockIdx.x % p.teams;
  const int member = blockIdx.x / p.teams;
  pdl_trigger();
  pdl_wait();  // queries, cache and metadata come from the kernels before

  // ---- this CTA's run of its team's tiles ----
  int64_t mine = 0;
  for (int b = threadIdx.x; b < p.num_seqs; b += kThreads) mine += team_tiles(p, b, team);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) scan[warp] = mine;
  if (threadIdx.x < 2) {  // no share left behind yet
    p.desc[(int64_t(blockIdx.x) * 2 + threadIdx.x) * 2] = make_int4(0, 0, 0, 0);
    if (threadIdx.x == 0) start[0] = p.num_seqs;
  }
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) total += scan[w];
  const int64_t per = (total + p.team_ctas - 1) / p.team_ctas;
  const int64_t begin = per * member;
  if (begin >= total) return;
  const int64_t count = min(per, total - begin);
  __syncthreads();
  int64_t carry = 0;
  for (int base = 0; base < p.num_seqs && carry <= begin; base += kThreads) {
    const int b = base + threadIdx.x;
    const int64_t c = b < p.num_seqs ? team_tiles(p, b, team) : 0;
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
      const Seq s = sequence(p, b);
      int64_t skip = begin - first;
      int g = team;
      while (skip >= group_tiles(p, s, g)) {
        skip -= group_tiles(p, s, g);
        g += p.teams;
      }
      start[0] = b;
      start[1] = g;
      start[2] = int(skip);
    }
    carry += sum;
    __syncthreads();
  }

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kQBufs; ++i) mbar_init(&bars[L::kQFull + i], 1), mbar_init(&bars[L::kQEmpty + i], 1);
    for (int i = 0; i < L::kRopeSlots; ++i) mbar_init(&bars[L::kRopeFull + i], 1), mbar_init(&bars[L::kRopeEmpty + i], 1);
    for (int i = 0; i < L::kPairSlots; ++i) mbar_init(&bars[L::kPairFull + i], 1), mbar_init(&bars[L::kPairEmpty + i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&bars[L::kSFull + i], 1), mbar_init(&bars[L::kSFree + i], kSmWarps);
    mbar_init(&bars[L::kPFull], kSmWarps);
    mbar_init(&bars[L::kPvDone], 1);
    mbar_init(&bars[L::kOFree], kSmWarps);
    mbar_init(&bars[L::kMmaDone], 2);
    mbar_init(&bars[L::kExch], kSmWarps);
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
  Walk walk = {start[0], start[1], start[2], count};
  Piece pc;

  if (warp == 0) {
    // ------------------------------ TMA producer ------------------------------
    if (lane == 0) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&ql_map)) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&qr_map)) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&c_map)) : "memory");
      const int rows = p.group_heads * p.group_tokens;
      const int sub_rows = p.sub_rows;
      const int sub_bytes = sub_rows * 128;
      uint32_t nq = 0, nt = 0, np = 0;  // query loads, rotary chunks and latent pairs issued
      bool ok = true;
      while (ok && walk.next(p, team, pc)) {
        const int qb = nq % L::kQBufs;
        uint64_t* const q_full = &bars[L::kQFull + qb];
        if (nq >= L::kQBufs && !mbar_wait(&bars[L::kQEmpty + qb], (nq / L::kQBufs - 1) & 1, p.err)) break;
        mbar_arrive_expect_tx(q_full, kChunks * rows * 128);
        const int head = pc.g % p.head_blocks * p.group_heads;
        const int tok = pc.s.q_begin + pc.g / p.head_blocks * p.group_tokens;
        const uint32_t qdst = sm + L::kQ + qb * L::kQBytes;
#pragma unroll 1
        for (int c = 0; c < kChunks - 1; ++c) tma_load_3d(qdst + c * N * 128, &ql_map, c * 64, head, tok, smem_u32(q_full));
        tma_load_3d(qdst + (kChunks - 1) * N * 128, &qr_map, 0, head, tok, smem_u32(q_full));
        ++nq;
        const int32_t* const bt = p.block_table + int64_t(pc.b) * p.bt_stride;
        for (int t = pc.t0; t < pc.t1 && ok; ++t) {
          const int valid = pc.valid(t);
          if (valid <= 0) break;
          const int subs = (valid + sub_rows - 1) / sub_rows;
          int page[kTile / 16], row[kTile / 16];
#pragma unroll
          for (int i = 0; i < kTile / 16; ++i) {
            if (i < subs) {
              const int at = t * kTile + i * sub_rows;
              const int lb = at / p.block_size;
              row[i] = at - lb * p.block_size;
              page[i] = __ldg(bt + lb);
              if (page[i] < 0 || page[i] >= p.num_blocks) {
                raise_device_error(p.err, NTB200_DEVERR_INDEX_RANGE);
                page[i] = -1;  // outside the map: the rows read as zeros
              }
            }
          }
          auto load = [&](uint32_t dst, int x, uint64_t* bar) {
#pragma unroll
            for (int i = 0; i < kTile / 16; ++i)
              if (i < subs) tma_load_3d(dst + i * sub_bytes, &c_map, x, row[i], page[i], smem_u32(bar));
          };
          const int rs = nt % L::kRopeSlots;
          if (nt >= L::kRopeSlots && !mbar_wait(&bars[L::kRopeEmpty + rs], (nt / L::kRopeSlots - 1) & 1, p.err)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&bars[L::kRopeFull + rs], subs * sub_bytes);
          load(sm + L::kRopeRing + rs * kChunkBytes, kLatent, &bars[L::kRopeFull + rs]);
          ++nt;
#pragma unroll 1
          for (int j = 0; j < kPairs; ++j) {
            const int ps = np % L::kPairSlots;
            if (np >= L::kPairSlots && !mbar_wait(&bars[L::kPairEmpty + ps], (np / L::kPairSlots - 1) & 1, p.err)) {
              ok = false;
              break;
            }
            mbar_arrive_expect_tx(&bars[L::kPairFull + ps], 2 * subs * sub_bytes);
            const uint32_t dst = sm + L::kPairRing + ps * kPairBytes;
            load(dst, j * 128, &bars[L::kPairFull + ps]);
            load(dst + kChunkBytes, j * 128 + 64, &bars[L::kPairFull + ps]);
            ++np;
          }
        }
      }
      // drain the copies that may still be in flight
      for (uint32_t i = nq > L::kQBufs ? nq - L::kQBufs : 0; i < nq; ++i)
        mbar_wait(&bars[L::kQFull + i % L::kQBufs], (i / L::kQBufs) & 1, p.err);
      for (uint32_t i = nt > L::kRopeSlots ? nt - L::kRopeSlots : 0; i < nt; ++i)
        mbar_wait(&bars[L::kRopeFull + i % L::kRopeSlots], (i / L::kRopeSlots) & 1, p.err);
      for (uint32_t i = np > L::kPairSlots ? np - L::kPairSlots : 0; i < np; ++i)
        mbar_wait(&bars[L::kPairFull + i % L::kPairSlots], (i / L::kPairSlots) & 1, p.err);
    }
  } else if (warp == 1) {
    // -------------------------- MMA issuer: S = Q C^T --------------------------
    if (lane == 0) {
      const uint32_t idesc = make_idesc(std::is_same<T, __nv_bfloat16>::value, 128, kTile);
      uint32_t nq = 0, nt = 0, np = 0, g = 0;
      bool ok = true;
      while (ok && walk.next(p, team, pc)) {
        const int qb = nq % L::kQBufs;
        if (!mbar_wait(&bars[L::kQFull + qb], (nq / L::kQBufs) & 1, p.err)) break;
        const uint32_t q = sm + L::kQ + qb * L::kQBytes;
        for (int t = pc.t0; t < pc.t1 && ok; ++t, ++g) {
          const int s = g & 1;
          // the softmax has read this buffer's scores of two tiles ago
          if (g >= 2 && !mbar_wait(&bars[L::kSFree + s], (g / 2 - 1) & 1, p.err)) {
            ok = false;
            break;
          }
          if (pc.valid(t) > 0) {
            const int rs = nt % L::kRopeSlots;
            if (!mbar_wait(&bars[L::kRopeFull + rs], (nt / L::kRopeSlots) & 1, p.err)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint64_t ar = sw128_kmajor_desc(q + (kChunks - 1) * N * 128);
            const uint64_t br = sw128_kmajor_desc(sm + L::kRopeRing + rs * kChunkBytes);
#pragma unroll
            for (int k = 0; k < 4; ++k) umma_f16(tmem + s * kTile, ar + 2 * k, br + 2 * k, idesc, k ? 1u : 0u);
            umma_commit(&bars[L::kRopeEmpty + rs]);
            ++nt;
#pragma unroll 1
            for (int j = 0; j < kPairs; ++j, ++np) {
              const int ps = np % L::kPairSlots;
              if (!mbar_wait(&bars[L::kPairFull + ps], (np / L::kPairSlots) & 1, p.err)) {
                ok = false;
                break;
              }
              tc_fence_after();
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint64_t a = sw128_kmajor_desc(q + (2 * j + h) * N * 128);
                const uint64_t b = sw128_kmajor_desc(sm + L::kPairRing + ps * kPairBytes + h * kChunkBytes);
#pragma unroll
                for (int k = 0; k < 4; ++k) umma_f16(tmem + s * kTile, a + 2 * k, b + 2 * k, idesc, 1u);
              }
            }
          }
          umma_commit(&bars[L::kSFull + s]);
        }
        umma_commit(&bars[L::kQEmpty + qb]);
        ++nq;
      }
      // every issued MMA completes before TMEM may be released
      umma_commit(&bars[L::kMmaDone]);
      mbar_wait(&bars[L::kMmaDone], 0, p.err);
    }
  } else if (warp == 2) {
    // ------------------------ MMA issuer: O^T += C^T P^T ------------------------
    if (lane == 0) {
      const uint32_t idesc = make_idesc(std::is_same<T, __nv_bfloat16>::value, 128, N) | (1u << 15);  // A MN-major
      uint32_t np = 0, g = 0, pieces = 0;
      bool ok = true;
      while (ok && walk.next(p, team, pc)) {
        for (int t = pc.t0; t < pc.t1 && ok; ++t, ++g) {
          // the first product of a piece overwrites O^T: the one before has been written out
          if (!mbar_wait(&bars[L::kPFull], g & 1, p.err) ||
              (t == pc.t0 && pieces >= 1 && !mbar_wait(&bars[L::kOFree], (pieces - 1) & 1, p.err))) {
            ok = false;
            break;
          }
          const int valid = pc.valid(t);
          if (valid > 0) {
            const int ks = (valid + 15) / 16;
            tc_fence_after();
            const uint64_t b = sw128_kmajor_desc(sm + L::kP);
#pragma unroll 1
            for (int j = 0; j < kPairs; ++j, ++np) {
              const int ps = np % L::kPairSlots;
              const uint32_t base = sm + L::kPairRing + ps * kPairBytes;
              for (int k = 0; k < ks; ++k)
                umma_f16(tmem + L::kTmemO + j * N, sw128_mnmajor_desc(base + k * 2048, kChunkBytes), b + 2 * k, idesc,
                         (t > pc.t0 || k > 0) ? 1u : 0u);
              umma_commit(&bars[L::kPairEmpty + ps]);
            }
          }
          umma_commit(&bars[L::kPvDone]);
        }
        ++pieces;
      }
      umma_commit(&bars[L::kMmaDone]);
      mbar_wait(&bars[L::kMmaDone], 0, p.err);
    }
  } else if (warp >= kFirstSmWarp) {
    // ------------------------------ softmax + output ------------------------------
    // Warp (quad, part): scores of rows 32 quad + lane at tokens 16 part .. + 16 (when the group
    // has such rows), and the block of O^T at latent columns 128 part + 32 quad + lane.  Every
    // warp holds the running max of all rows (lane's and lane + 32's), so all agree on when to
    // rescale without another exchange.
    constexpr int kRowRegs = N == 64 ? 2 : 1;
    const int quad = warp & 3;
    const int part = (warp - kFirstSmWarp) >> 2;
    const int r = quad * 32 + lane;
    const bool active = quad * 32 < N;
    const uint32_t lanes = uint32_t(quad * 32) << 16;
    const uint32_t o_tmem = tmem + L::kTmemO + part * N + lanes;
    uint64_t* const exch = &bars[L::kExch];
    uint32_t uses = 0;
    // Publishes an active thread's value for its row and leaves every row's four in `red`.
    auto exchange = [&](float v) -> const float* {
      float* const buf = red + (uses & 1) * (kParts * kMaxRows);
      if (active) buf[part * kMaxRows + r] = v;
      __syncwarp();
      if (lane == 0) mbar_arrive(exch);
      const bool got = mbar_wait_warp(exch, uses & 1, p.err);
      ++uses;
      return got ? buf : nullptr;
    };
    uint32_t g = 0, np = 0, pieces = 0;
    bool ok = true;
    while (ok && walk.next(p, team, pc)) {
      const int tok0 = pc.g / p.head_blocks * p.group_tokens;
      const int head0 = pc.g % p.head_blocks * p.group_heads;
      // rows of the group: (token, head) = (row / group_heads, row % group_heads)
      auto row_there = [&](int row, int& tok, int& head) {
        const int rt = row / p.group_heads;
        tok = tok0 + rt;
        head = head0 + row - rt * p.group_heads;
        return rt < p.group_tokens && tok < pc.s.q_len && head < p.num_heads;
      };
      int tok, head;
      const bool there = row_there(r, tok, head);
      // this row sees keys [0, limit)
      const int limit = there && active ? max(pc.s.ctx - pc.s.q_len + tok + 1, 0) : 0;
      float m[kRowRegs];
#pragma unroll
      for (int i = 0; i < kRowRegs; ++i) m[i] = -INFINITY;
      float l_run = 0.f;
      for (int t = pc.t0; t < pc.t1; ++t, ++g) {
        const int s = g & 1;
        const int valid = pc.valid(t);
        if (!mbar_wait_warp(&bars[L::kSFull + s], (g / 2) & 1, p.err)) {
          ok = false;
          break;
        }
        tc_fence_after();
        float x[kPartCols];
        float mx = -INFINITY;
        if (active) {
          uint32_t v[kPartCols];
          __syncwarp();
          tmem_ld_16(tmem + lanes + s * kTile + part * kPartCols, v);
          const int seen = limit - t * kTile - part * kPartCols;
#pragma unroll
          for (int i = 0; i < kPartCols; ++i) {
            x[i] = i < seen ? __uint_as_float(v[i]) * p.scale_log2 : -INFINITY;
            mx = fmaxf(mx, x[i]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[L::kSFree + s]);
        const float* const all = exchange(mx);
        if (all == nullptr) {
          ok = false;
          break;
        }
        float alpha[kRowRegs];
        bool grow = false;
#pragma unroll
        for (int i = 0; i < kRowRegs; ++i) {
          const int row = lane + 32 * i;
          float m_new = m[i];
#pragma unroll
          for (int q = 0; q < kParts; ++q)
            if (row < N) m_new = fmaxf(m_new, all[q * kMaxRows + row]);
          const bool up = m_new > m[i] + kRescaleLog2;  // also true for the first finite max
          alpha[i] = up ? hw_exp2(m[i] - m_new) : 1.f;
          if (up) m[i] = m_new;
          grow = grow || up;
        }
        const bool any = __any_sync(0xffffffffu, grow);
        uint32_t pk[kPartCols / 2];
        if (active) {
          const float mine_m = kRowRegs == 2 && quad == 1 ? m[kRowRegs - 1] : m[0];
          const float mine_a = kRowRegs == 2 && quad == 1 ? alpha[kRowRegs - 1] : alpha[0];
          const float m_use = mine_m == -INFINITY ? 0.f : mine_m - kBias<T>;
          l_run *= mine_a;
          float l2[2] = {0.f, 0.f};
#pragma unroll
          for (int i = 0; i < kPartCols / 2; ++i) {
            const float p0 = hw_exp2(x[2 * i] - m_use);
            const float p1 = hw_exp2(x[2 * i + 1] - m_use);
            l2[i & 1] += p0 + p1;
            Pair<T>::store(reinterpret_cast<T*>(&pk[i]), p0, p1);
          }
          l_run += l2[0] + l2[1];
        }
        // P and O^T are free once the product of the tile before is complete
        if (g >= 1 && !mbar_wait_warp(&bars[L::kPvDone], (g - 1) & 1, p.err)) {
          ok = false;
          break;
        }
        if (any && t > pc.t0) {
          tc_fence_after();
#pragma unroll
          for (int c0 = 0; c0 < N; c0 += 16) {
            uint32_t v[16];
            __syncwarp();
            tmem_ld_16(o_tmem + c0, v);
#pragma unroll
            for (int c = 0; c < 16; ++c) {
              const float a = __shfl_sync(0xffffffffu, alpha[(c0 + c) / 32], (c0 + c) % 32);
              v[c] = __float_as_uint(__uint_as_float(v[c]) * a);
            }
            tmem_st_16(o_tmem + c0, v);
          }
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        }
        if (active && r < N) {
          // P [row, token], 128-byte swizzled rows; this part's 16 tokens are two 16-byte units
          uint8_t* const prow = smem + L::kP + r * 128;
#pragma unroll
          for (int i = 0; i < 2; ++i)
            *reinterpret_cast<uint4*>(prow + (((part * 2 + i) ^ (r & 7)) << 4)) =
                make_uint4(pk[4 * i], pk[4 * i + 1], pk[4 * i + 2], pk[4 * i + 3]);
        }
        if (valid > 0) {
          if (valid & 15) {
            // rows past the last visible key, up to the product's next step of 16, hold whatever
            // memory held there: zeroed, so that P = 0 never meets a non-finite value
            const int t0 = valid, n = 16 - (valid & 15);
            for (int i = threadIdx.x - 32 * kFirstSmWarp; i < n * 64; i += 32 * kSmWarps) {
              const int c = (i >> 3) & 7;  // chunk
              const uint32_t ps = (np + (c >> 1)) % L::kPairSlots;
              *reinterpret_cast<uint4*>(smem + L::kPairRing + ps * kPairBytes + (c & 1) * kChunkBytes +
                                        (t0 + (i >> 6)) * 128 + (i & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
          }
          np += kPairs;
        }
        fence_proxy_async_smem();  // P and the zeros -> tensor core
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[L::kPFull]);
      }
      if (!ok) break;
      // O^T is final once the piece's last product is complete
      ok = mbar_wait_warp(&bars[L::kPvDone], (g - 1) & 1, p.err);
      const float* const all = ok ? exchange(l_run) : nullptr;
      if (all == nullptr) {
        ok = false;
        break;
      }
      tc_fence_after();
      const bool whole = pc.t0 == 0 && pc.t1 == pc.n;
      const int64_t share = int64_t(blockIdx.x) * 2 + (pieces > 0 ? 1 : 0);
      float inv[kRowRegs];
      int64_t dst[kRowRegs];  // element offset of the row's output, -1: no such row
#pragma unroll
      for (int i = 0; i < kRowRegs; ++i) {
        const int row = lane + 32 * i;
        float l = 0.f;
        if (row < N)
#pragma unroll
          for (int q = 0; q < kParts; ++q) l += all[q * kMaxRows + row];
        inv[i] = l == 0.f ? 0.f : 1.f / l;
        int rtok, rhead;
        const bool rthere = row_there(row, rtok, rhead) && row < N;
        const float lse2 = l == 0.f ? -INFINITY : m[i] - kBias<T> + log2f(l);
        if (whole) {
          dst[i] = rthere ? int64_t(pc.s.q_begin + rtok) * p.o_tok + int64_t(rhead) * p.o_head : -1;
          if (rthere && p.lse != nullptr && quad == 0 && part == 0)
            p.lse[int64_t(pc.s.q_begin + rtok) * p.lse_tok + rhead] = lse2 * 0.6931471805599453f;
        } else {
          dst[i] = rthere ? (share * kMaxRows + row) * kLatent : -1;
          if (rthere && quad == 0 && part == 0) p.part_lse[share * kMaxRows + row] = lse2;
        }
      }
      if (!whole && quad == 0 && part == 0 && lane == 0) {
        p.desc[share * 2] = make_int4(1, pc.t0, pc.t1, pc.n);
        p.desc[share * 2 + 1] = make_int4(pc.s.q_begin + tok0, pc.s.q_len - tok0, head0, 0);
      }
      const int col = part * 128 + quad * 32 + lane;
#pragma unroll
      for (int c0 = 0; c0 < N; c0 += 16) {
        uint32_t v[16];
        __syncwarp();
        tmem_ld_16(o_tmem + c0, v);
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          const float k = __shfl_sync(0xffffffffu, inv[(c0 + c) / 32], (c0 + c) % 32);
          const int64_t at = __shfl_sync(0xffffffffu, dst[(c0 + c) / 32], (c0 + c) % 32);
          if (at < 0) continue;
          const float o = k == 0.f ? 0.f : __uint_as_float(v[c]) * k;  // an empty row's O^T was never written
          if (whole) static_cast<T*>(p.out)[at + col] = Elem<T>::from_f(o);
          else p.part_o[at + col] = o;
        }
      }
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

// Joins the shares of every item that was cut.  The CTA whose first piece ends an item (its
// share 0 has t0 > 0 and t1 = n) names that item; the shares before it are the last ones of
// the CTAs before, back to the one that starts at tile 0.
constexpr int kJoinThreads = kLatent / 4;
constexpr int kJoinRows = 4;  // rows a CTA

template <typename T>
__global__ void __launch_bounds__(kJoinThreads) latent_join_kernel(const LatentParams p) {
  __shared__ int list[1024];  // shares of the item
  pdl_trigger();
  pdl_wait();
  const int cta = blockIdx.x;
  const int4 end = p.desc[int64_t(cta) * 4];
  if (end.x == 0 || end.y == 0 || end.z != end.w) return;
  const int4 where = p.desc[int64_t(cta) * 4 + 1];
  __shared__ int num;
  if (threadIdx.x == 0) {
    int n = 0;
    list[n++] = cta * 2;
    for (int c = cta - p.teams; c >= 0 && n < 1024; c -= p.teams) {
      const int share = c * 2 + (p.desc[int64_t(c) * 4 + 2].x != 0 ? 1 : 0);
      list[n++] = share;
      if (p.desc[int64_t(share) * 2].y == 0) break;
    }
    num = n;
  }
  __syncthreads();
  const int n = num;
  for (int r = blockIdx.y * kJoinRows; r < (int(blockIdx.y) + 1) * kJoinRows; ++r) {
    const int tok = r / p.group_heads;
    const int head = where.z + r - tok * p.group_heads;
    if (tok >= p.group_tokens || tok >= where.y || head >= p.num_heads) continue;
    float top = -INFINITY;
    for (int i = 0; i < n; ++i) top = fmaxf(top, p.part_lse[int64_t(list[i]) * kMaxRows + r]);
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const int64_t row = int64_t(list[i]) * kMaxRows + r;
      const float w = exp2f(p.part_lse[row] - ref);
      const float4 o = reinterpret_cast<const float4*>(p.part_o + row * kLatent)[threadIdx.x];
      sum += w;
      acc.x += w * o.x, acc.y += w * o.y, acc.z += w * o.z, acc.w += w * o.w;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const float y[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
    T* const o = static_cast<T*>(p.out) + int64_t(where.x + tok) * p.o_tok + int64_t(head) * p.o_head;
    *reinterpret_cast<Vec<T, 4>*>(o + threadIdx.x * 4) = pack_f<T, 4>(y);
    if (p.lse != nullptr && threadIdx.x == 0)
      p.lse[int64_t(where.x + tok) * p.lse_tok + head] =
          sum == 0.f ? -INFINITY : (ref + log2f(sum)) * 0.6931471805599453f;
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

// the cache [blocks, block_size, 576]: box = sub_rows tokens of a page x 64 columns
int make_cache_map(CUtensorMap* map, const void* base, bool bf16, int64_t blocks, int64_t block_size,
                   int64_t block_stride, int64_t page_stride, int sub_rows) {
  EncodeTiledFn enc = encode_fn();
  if (enc == nullptr) return fail(NTB200_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const cuuint64_t dims[3] = {cuuint64_t(kLatent + kRope), cuuint64_t(block_size), cuuint64_t(blocks)};
  const cuuint64_t strides[2] = {cuuint64_t(page_stride * 2),
                                 cuuint64_t((blocks > 1 ? block_stride : block_size * page_stride) * 2)};
  const cuuint32_t box[3] = {64, cuuint32_t(sub_rows), 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
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
  const int rows = p.group_heads * p.group_tokens;
  return launch_kernel("latent_attention (join)", latent_join_kernel<T>,
                       dim3(ctas, unsigned(ceil_div(rows, kJoinRows))), dim3(kJoinThreads), 0, s, p);
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
constexpr int kMaxCtas = 1024;

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
  if (query_start_loc == nullptr && num_seqs > 0 && num_tokens % num_seqs != 0)
    return fail(NTB200_ERR_INVALID_ARGUMENT, "latent_attention: without query_start_loc every sequence has num_tokens / num_seqs queries");
  if (num_seqs == 0 || num_tokens == 0 || (query_start_loc != nullptr && max_query_len == 0)) return NTB200_OK;
  if (num_seqs > 0x7fffffff || num_tokens > 0x7fffffff || num_heads > 65535 || num_blocks > 0x7fffffff ||
      max_blocks_per_seq > 0x7fffffff / block_size)
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
  p.sub_rows = block_size % 64 == 0 ? 64 : block_size % 32 == 0 ? 32 : 16;
  p.num_blocks = int(num_blocks);
  p.max_blocks = int(max_blocks_per_seq);
  p.head_blocks = int(ceil_div(num_heads, kMaxRows));
  p.group_heads = int(ceil_div(num_heads, p.head_blocks));
  p.group_tokens = std::min(kMaxRows / p.group_heads, p.max_query);
  p.scale_log2 = scale * 1.4426950408889634f;  // softmax in the exp2 domain
  p.err = device_error_word();
  const int64_t groups = ceil_div(p.max_query, p.group_tokens) * p.head_blocks;
  p.teams = groups <= kMaxTeams ? int(groups) : 1;
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
    st = make_cache_map(&c, kv_cache, bf16, num_blocks, block_size, cache_block_stride, cache_page_stride, p.sub_rows);
    if (st != NTB200_OK) return st;
  } else {
    c = ql;  // never read: every context is empty
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return bf16 ? by_rows<__nv_bfloat16>(ql, qr, c, p, 128, s) : by_rows<__half>(ql, qr, c, p, 131, s);
}
