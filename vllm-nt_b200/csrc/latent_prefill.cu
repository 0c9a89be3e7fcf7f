// Latent attention with the keys and values of every head expanded from the latent (prompts):
//   s[i, j] = scale * (q_nope[i] . k_nope[j, h] + q_rope[i] . k_rope[j]),
//   out[i, h] = sum_j softmax(s[i])_j v[j, h],   lse[i, h] = ln sum_j exp(s[i, j])
// over each sequence's keys, causal masking aligned to their end.  q [tokens, heads, 192] is
// [nope (128) | rope (64)]; the rotary key is one row a token for all heads and is read as it
// is, never copied to the heads.
//
// Persistent, one CTA per SM, 384 threads.  A work item is 256 query rows of one head, as two
// 128-row tiles A and B that share every K and V tile (128 keys) brought in:
//   warps 0-3, 4-7  softmax of tile A, B: one thread a row, whose 128 scores it takes into
//                   registers at once (208 a thread, drawn from the issuing warps'), so that one
//                   S buffer serves both tiles and the next product runs while this one's softmax
//                   does; the running maximum is refreshed only when it grows by over 2^8 (the
//                   output is rescaled then); weights go to TMEM, rounded to the type.
//   warp 8          S = Q K^T of A and B in turn (tcgen05, M = N = 128, twelve steps of 16).
//   warp 9          O += P V (P from TMEM, V as it lies, MN-major, in two halves of 64 columns).
//   warp 10         TMA: Q tiles and a ring of eight 16 KB chunks (128 rows x 64 columns), K_j+1
//                   ahead of V_j, as S runs a tile ahead of P V.
// TMEM: S 128 columns, P_A and P_B 64 each, O_A and O_B 128 each.  Items are dealt to and fro over
// the CTAs, a sequence's last (longest) rows first.
// Bound: tensor core, 2 * 320 operations a visible (query, key) pair.  A causal prompt of 8192
// tokens and 32 heads takes 540 to 556 us, 1250 TFLOP/s, in a short run at 1.68 GHz, and 640 us, 1080
// TFLOP/s, where calls follow each other for long: it draws the power limit, which then leaves 1.44 GHz
// (635 us in a short run with an S buffer a tile that also held its
// weights, which kept a tile's next product waiting for P V).
#include <algorithm>

#include "common.cuh"
#include "latent_ring.cuh"
#include "tcgen05.cuh"

namespace ntb200 {
namespace {

constexpr int kNope = 128, kRope = 64, kV = 128;
constexpr int kQChunks = (kNope + kRope) / 64;  // 64-column chunks of a query or key row
constexpr int kVChunks = kV / 64;
constexpr int kBQ = 128, kBK = 128;
constexpr int kItemRows = 2 * kBQ;
constexpr int kChunkBytes = 128 * 128;  // 128 rows x 64 columns
constexpr int kRing = 8;
constexpr int kThreads = 384;
constexpr int kSWarp = 8, kPvWarp = 9, kTmaWarp = 10, kAllocWarp = 11;
constexpr float kRescaleLog2 = 8.0f;
// registers: launched with 168 a thread, the two softmax warpgroups draw what the third gives up
constexpr int kSoftmaxRegs = 208, kIssueRegs = 88;
static_assert(256 * kSoftmaxRegs + 128 * kIssueRegs <= 384 * 168, "register split");
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kTmemP = 128;  // S at 0; P_A, P_B at 128, 192
constexpr uint32_t kTmemO = 256;  // O_A, O_B at 256, 384

static_assert(kQChunks == kRingKeys && kVChunks == kRingValues && kRing == kRingChunks, "the ring's order");

struct Smem {
  static constexpr int kQ = 0;  // [2 tiles][3 chunks]
  static constexpr int kKv = kQ + 2 * kQChunks * kChunkBytes;
  static constexpr int kBars = kKv + kRing * kChunkBytes;
  // indexes of the mbarriers: one of each for tile A and B, or for even and odd key tiles
  static constexpr int kQFull = 0, kQEmpty = 2, kKFull = 4, kKEmpty = 6, kVFull = 8, kVEmpty = 10, kSFull = 12,
                       kPFull = 14, kPvDone = 16, kOFree = 18, kSFree = 20, kMmaDone = 21, kKDone = 22, kNumBars = 24;
  static constexpr int kTmemBase = kBars + 8 * kNumBars;
  static constexpr int kRow = kTmemBase + 16;  // [256 rows] int2: where a softmax thread's output goes
  static constexpr int kBytes = kRow + kItemRows * 8;
};
static_assert(Smem::kBytes <= 227 * 1024, "shared memory");

struct PrefillParams {
  void* out;
  float* lse;
  const int32_t *cu_q, *cu_k;
  int64_t o_tok, o_head, lse_tok;
  int num_seqs, num_q, num_k, num_heads;
  int causal;
  float scale_log2;
  unsigned int* err;
};

// 256 rows of one head: tile x has rows q0 + 128 x .. of the sequence (rows[x] of them) and
// visits tiles[x] key tiles.
struct Item {
  int head, q_begin, q_len, k_begin, ctx, q0;
  int rows[2], tiles[2];
};

// Walks a CTA's items (every role walks the same).  A warp holds 32 sequences' item counts at a
// time and steps through the list as the item number grows.
struct Walk {
  int base;    // first sequence of the 32 held
  int before;  // items of the sequences before them
  int upto;    // this lane's inclusive count within the 32
  int q_begin, q_len, k_begin, ctx;
  bool broken;  // cu_q fell somewhere before: the sequences behind could overlap, and are left out

  __device__ __forceinline__ void load(const PrefillParams& p, int first) {
    const int lane = threadIdx.x & 31;
    const int b = first + lane;
    base = first;
    q_begin = q_len = k_begin = ctx = 0;
    bool fall = false;
    if (b < p.num_seqs) {
      q_begin = p.cu_q[b];
      k_begin = p.cu_k[b];
      const int q_end = p.cu_q[b + 1], k_end = p.cu_k[b + 1];
      fall = q_end < q_begin;
      // (compared, not subtracted: the difference of far locations wraps)
      if (q_begin < 0 || fall || q_end > p.num_q || k_begin < 0 || k_end < k_begin || k_end > p.num_k) {
        raise_device_error(p.err, NTB200_DEVERR_INDEX_RANGE);
        q_begin = k_begin = 0;
      } else {
        q_len = q_end - q_begin;
        ctx = k_end - k_begin;
      }
    }
    const unsigned falls = __ballot_sync(0xffffffffu, fall);
    if (broken || (falls & ((1u << lane) - 1)) != 0) q_begin = q_len = k_begin = ctx = 0;
    broken = broken || falls != 0;
    upto = (q_len + kItemRows - 1) / kItemRows * p.num_heads;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
  }

  __device__ __forceinline__ void begin(const PrefillParams& p) {
    before = 0;
    broken = false;
    load(p, 0);
  }

  // item w (growing from call to call); false past the last one
  __device__ __forceinline__ bool get(const PrefillParams& p, int w, Item& it) {
    for (;;) {
      const int all = __shfl_sync(0xffffffffu, upto, 31);
      if (w < before + all) break;
      if (base + 32 >= p.num_seqs) return false;
      before += all;
      load(p, base + 32);
    }
    const unsigned past = __ballot_sync(0xffffffffu, w < before + upto);
    const int at = __ffs(past) - 1;
    const int below = __shfl_sync(0xffffffffu, upto, at > 0 ? at - 1 : 0);
    const int prior = at > 0 ? below : 0;
    it.q_begin = __shfl_sync(0xffffffffu, q_begin, at);
    it.q_len = __shfl_sync(0xffffffffu, q_len, at);
    it.k_begin = __shfl_sync(0xffffffffu, k_begin, at);
    it.ctx = __shfl_sync(0xffffffffu, ctx, at);
    const int i = w - before - prior;
    const int block = i / p.num_heads;
    it.head = i - block * p.num_heads;
    const int blocks = (it.q_len + kItemRows - 1) / kItemRows;
    it.q0 = (blocks - 1 - block) * kItemRows;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int first = it.q0 + x * kBQ;
      it.rows[x] = min(max(it.q_len - first, 0), kBQ);
      const int last = it.ctx - it.q_len + first + it.rows[x];
      const int keys = it.rows[x] == 0 ? 0 : p.causal ? min(max(last, 0), it.ctx) : it.ctx;
      it.tiles[x] = (keys + kBK - 1) / kBK;
    }
    return true;
  }
};

// The ring's operations as the producer's warp makes them (see RingFill).  A wait for key tile g is one for
// phase g / 2 of barrier g & 1.
struct RingOps {
  uint64_t* bars;
  uint32_t ring;  // its shared-memory address
  const CUtensorMap *kn_map, *kr_map, *v_map;
  uint32_t elected;
  unsigned int* err;
  int k_head, k_row, v_head, v_row;  // of the next keys and values

  __device__ __forceinline__ bool wait(int bar, uint32_t g) {
    return mbar_wait_warp(&bars[bar + (g & 1)], (g / 2) & 1, err);
  }
  __device__ __forceinline__ bool keys_half_used(uint32_t g) { return wait(Smem::kKEmpty, g); }
  __device__ __forceinline__ bool keys_used(uint32_t g) { return wait(Smem::kKDone, g); }
  __device__ __forceinline__ bool values_used(uint32_t g) { return wait(Smem::kVEmpty, g); }
  __device__ __forceinline__ void load_keys(uint32_t g) {
    if (elected) {
      uint64_t* const full = &bars[Smem::kKFull + (g & 1)];
      mbar_arrive_expect_tx(full, kQChunks * kChunkBytes);
      for (int c = 0; c < kQChunks; ++c) {
        const uint32_t dst = ring + (k_chunk(g) + c) % kRing * kChunkBytes;
        if (c < kNope / 64) tma_load_3d(dst, kn_map, c * 64, k_head, k_row, smem_u32(full));
        else tma_load_2d(dst, kr_map, 0, k_row, smem_u32(full));
      }
    }
    __syncwarp();
  }
  __device__ __forceinline__ void load_values(uint32_t g) {
    if (elected) {
      uint64_t* const full = &bars[Smem::kVFull + (g & 1)];
      mbar_arrive_expect_tx(full, kVChunks * kChunkBytes);
      for (int c = 0; c < kVChunks; ++c)
        tma_load_3d(ring + (v_chunk(g) + c) % kRing * kChunkBytes, v_map, c * 64, v_head, v_row, smem_u32(full));
    }
    __syncwarp();
  }
};

// A CTA's k-th item.  Rounds go over the CTAs to and fro: within a sequence items shrink, and dealt
// in one direction the first CTA would have the larger item of every round (8192 tokens of 32
// heads: 14% over the mean, so 2%).
__device__ __forceinline__ int item_of(int k) {
  return k * int(gridDim.x) + int((k & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
}

// 32 TMEM columns on their way into registers, which are there once tmem_ld_done has named them.
__device__ __forceinline__ void tmem_ld_32_begin(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_done(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])::"memory");
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
    latent_prefill_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap kn_map,
                          const __grid_constant__ CUtensorMap kr_map, const __grid_constant__ CUtensorMap v_map,
                          const PrefillParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sm = smem_u32(smem);
  uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + Smem::kBars);
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(smem + Smem::kTmemBase);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars[Smem::kQFull + i], 1);
      mbar_init(&bars[Smem::kQEmpty + i], 1);
      mbar_init(&bars[Smem::kKFull + i], 1);
      mbar_init(&bars[Smem::kKEmpty + i], 1);
      mbar_init(&bars[Smem::kKDone + i], 1);
      mbar_init(&bars[Smem::kVFull + i], 1);
      mbar_init(&bars[Smem::kVEmpty + i], 1);
      mbar_init(&bars[Smem::kSFull + i], 1);
      mbar_init(&bars[Smem::kPFull + i], 4);  // one arrive a softmax warp
      mbar_init(&bars[Smem::kPvDone + i], 1);
      mbar_init(&bars[Smem::kOFree + i], 4);
    }
    mbar_init(&bars[Smem::kSFree], 4);
    mbar_init(&bars[Smem::kMmaDone], 2);
    fence_mbar_init();
  }
  pdl_wait();  // queries, keys and metadata come from the kernels before
  if (warp == kAllocWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  Walk walk;
  Item it;
  walk.begin(p);

  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
  if (warp == kTmaWarp) {
    // ------------------------------ TMA producer ------------------------------
    const uint32_t elected = elect_one();
    if (elected) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&q_map)) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&kn_map)) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&kr_map)) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&v_map)) : "memory");
    }
    __syncwarp();
    uint32_t nq[2] = {0, 0};  // Q tiles loaded
    RingOps ops = {bars, sm + Smem::kKv, &kn_map, &kr_map, &v_map, elected, p.err, 0, 0, 0, 0};
    RingFill fill;
    bool ok = true;
    for (int k = 0; ok && walk.get(p, item_of(k), it); ++k) {
      auto load_q = [&](int x) {
        if (!ok || it.tiles[x] == 0) return;
        uint64_t* const full = &bars[Smem::kQFull + x];
        if (nq[x] >= 1) ok = mbar_wait_warp(&bars[Smem::kQEmpty + x], (nq[x] - 1) & 1, p.err);
        if (!ok) return;
        if (elected) {
          mbar_arrive_expect_tx(full, kQChunks * kChunkBytes);
          for (int c = 0; c < kQChunks; ++c)
            tma_load_3d(sm + Smem::kQ + (x * kQChunks + c) * kChunkBytes, &q_map, c * 64, it.head,
                        it.q_begin + it.q0 + x * kBQ, smem_u32(full));
        }
        __syncwarp();
        ++nq[x];
      };
      const int tiles = max(it.tiles[0], it.tiles[1]);
      load_q(0);
      for (int j = 0; ok && j < tiles; ++j) {
        ops.k_head = it.head;
        ops.k_row = it.k_begin + j * kBK;
        ok = fill.keys(ops);
        if (j == 0) load_q(1);
        ok = ok && fill.values_behind(ops);
        ops.v_head = ops.k_head;
        ops.v_row = ops.k_row;
      }
    }
    ok = ok && fill.last_values(ops);
    // drain the copies that may still be in flight
    for (int x = 0; x < 2; ++x)
      if (nq[x] > 0) mbar_wait_warp(&bars[Smem::kQFull + x], (nq[x] - 1) & 1, p.err);
    for (uint32_t g = fill.nk > 2 ? fill.nk - 2 : 0; g < fill.nk; ++g) ops.wait(Smem::kKFull, g);
    for (uint32_t g = fill.nv > 2 ? fill.nv - 2 : 0; g < fill.nv; ++g) ops.wait(Smem::kVFull, g);
  } else if (warp == kSWarp) {
    // -------------------------- MMA issuer: S = Q K^T --------------------------
    const uint32_t elected = elect_one();
    const uint32_t idesc = make_idesc(std::is_same<T, __nv_bfloat16>::value, kBQ, kBK);
    uint32_t nq[2] = {0, 0};
    uint32_t g = 0, ns = 0;  // key tiles passed, products issued
    bool ok = true;
    for (int k = 0; ok && walk.get(p, item_of(k), it); ++k) {
      const int tiles = max(it.tiles[0], it.tiles[1]);
      for (int j = 0; ok && j < tiles; ++j, ++g) {
        // what is usually there comes first: a wait that is already over costs over 100 cycles too
        ok = mbar_wait_warp(&bars[Smem::kKFull + (g & 1)], (g / 2) & 1, p.err);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (!ok || j >= it.tiles[x]) continue;
          const bool last_user = x == 1 || j >= it.tiles[1];
          // the product before is in its warps' registers
          ok = (j > 0 || mbar_wait_warp(&bars[Smem::kQFull + x], nq[x] & 1, p.err)) &&
               (ns == 0 || mbar_wait_warp(&bars[Smem::kSFree], (ns - 1) & 1, p.err));
          if (!ok) continue;
          tc_fence_after();
          const uint64_t a0 = sw128_kmajor_desc(sm + Smem::kQ + x * kQChunks * kChunkBytes);
          const uint64_t b0 = sw128_kmajor_desc(sm + Smem::kKv);
#pragma unroll
          for (int c = 0; c < kQChunks; ++c) {
            const uint32_t s = (k_chunk(g) + c) % kRing;
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_elected(tmem, a0 + c * (kChunkBytes >> 4) + 2 * k, b0 + s * (kChunkBytes >> 4) + 2 * k, idesc,
                           (c | k) ? 1u : 0u, elected);
            if (last_user && c == 1) commit_elected(&bars[Smem::kKEmpty + (g & 1)], elected);
          }
          commit_elected(&bars[Smem::kSFull + x], elected);
          if (last_user) commit_elected(&bars[Smem::kKDone + (g & 1)], elected);
          ++ns;
          if (j + 1 == it.tiles[x]) {
            commit_elected(&bars[Smem::kQEmpty + x], elected);
            ++nq[x];
          }
        }
      }
    }
    // every issued MMA completes before TMEM may be released
    commit_elected(&bars[Smem::kMmaDone], elected);
    mbar_wait_warp(&bars[Smem::kMmaDone], 0, p.err);
  } else if (warp == kPvWarp) {
    // -------------------------- MMA issuer: O += P V --------------------------
    const uint32_t elected = elect_one();
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    const uint32_t idesc = make_idesc(kBf16, kBQ, kV) | (1u << 16);       // B (V) MN-major
    const uint32_t idesc_half = make_idesc(kBf16, kBQ, 64) | (1u << 16);  // one chunk of it
    uint32_t np[2] = {0, 0};     // products issued a tile
    uint32_t items[2] = {0, 0};  // outputs begun
    uint32_t g = 0;              // key tiles passed
    bool ok = true;
    for (int k = 0; ok && walk.get(p, item_of(k), it); ++k) {
      const int tiles = max(it.tiles[0], it.tiles[1]);
      for (int j = 0; ok && j < tiles; ++j, ++g) {
        const int inside = min(it.ctx - j * kBK, kBK);  // rows of this V tile that belong to the sequence
        const int steps = (inside + 15) / 16;
        const uint32_t s0 = v_chunk(g) % kRing, s1 = (v_chunk(g) + 1) % kRing;
        const uint64_t v0 = sw128_mnmajor_desc(sm + Smem::kKv + s0 * kChunkBytes, kChunkBytes);
        const uint64_t v1 = sw128_mnmajor_desc(sm + Smem::kKv + s1 * kChunkBytes, kChunkBytes);
        ok = mbar_wait_warp(&bars[Smem::kVFull + (g & 1)], (g / 2) & 1, p.err);
        if (ok && (inside & 15) != 0) {
          // rows behind the sequence, up to the product's last step of 16, are another's: zeroed,
          // so that a weight of 0 never meets a non-finite value
          for (int i = lane; i < (steps * 16 - inside) * 8 * kVChunks; i += 32)
            *reinterpret_cast<uint4*>(smem + Smem::kKv + ((i & 8) ? s1 : s0) * kChunkBytes + (inside + (i >> 4)) * 128 +
                                      (i & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
          fence_proxy_async_smem();
          __syncwarp();
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (!ok || j >= it.tiles[x]) continue;
          const bool last_user = x == 1 || j >= it.tiles[1];
          ok = (j > 0 || items[x] == 0 || mbar_wait_warp(&bars[Smem::kOFree + x], (items[x] - 1) & 1, p.err)) &&
               mbar_wait_warp(&bars[Smem::kPFull + x], np[x] & 1, p.err);
          if (!ok) continue;
          tc_fence_after();
          const uint32_t o_tmem = tmem + kTmemO + x * kV, p_tmem = tmem + kTmemP + x * (kBK / 2);
          if (s1 == s0 + 1) {  // both chunks of V lie together: one product over 128 columns
#pragma unroll
            for (int k = 0; k < kBK / 16; ++k)
              if (k < steps) umma_tmem_a_elected(o_tmem, p_tmem + k * 8, v0 + k * (2048 >> 4), idesc, (j > 0 || k > 0) ? 1u : 0u, elected);
          } else {             // the ring wraps between them
#pragma unroll
            for (int k = 0; k < kBK / 16; ++k)
              if (k < steps) {
                umma_tmem_a_elected(o_tmem, p_tmem + k * 8, v0 + k * (2048 >> 4), idesc_half, (j > 0 || k > 0) ? 1u : 0u, elected);
                umma_tmem_a_elected(o_tmem + 64, p_tmem + k * 8, v1 + k * (2048 >> 4), idesc_half, (j > 0 || k > 0) ? 1u : 0u, elected);
              }
          }
          commit_elected(&bars[Smem::kPvDone + x], elected);
          if (last_user) commit_elected(&bars[Smem::kVEmpty + (g & 1)], elected);
          ++np[x];
          if (j == 0) ++items[x];
        }
      }
    }
    commit_elected(&bars[Smem::kMmaDone], elected);
    mbar_wait_warp(&bars[Smem::kMmaDone], 0, p.err);
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ------------------------------ softmax + output ------------------------------
    const int x_tile = warp >> 2;
    const int r = (warp & 3) * 32 + lane;
    const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
    const uint32_t s_tmem = tmem + lanes;
    const uint32_t p_tmem = tmem + kTmemP + x_tile * (kBK / 2) + lanes;
    const uint32_t o_tmem = tmem + kTmemO + x_tile * kV + lanes;
    int2* const row_of = reinterpret_cast<int2*>(smem + Smem::kRow) + threadIdx.x;
    uint32_t g = 0;  // this tile's key tiles done
    bool ok = true;
    for (int k = 0; ok && walk.get(p, item_of(k), it); ++k) {
      const int tiles = x_tile == 0 ? it.tiles[0] : it.tiles[1];
      // this row sees keys [0, limit)
      const int ctx = it.ctx;
      const bool there = r < (x_tile == 0 ? it.rows[0] : it.rows[1]);
      *row_of = make_int2(there ? it.q_begin + it.q0 + x_tile * kBQ + r : -1, it.head);  // (not held through the tiles)
      const int limit = !there ? 0
                        : p.causal ? min(max(ctx - it.q_len + it.q0 + x_tile * kBQ + r + 1, 0), ctx)
                                   : ctx;
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < tiles; ++j, ++g) {
        if (!mbar_wait_warp(&bars[Smem::kSFull + x_tile], g & 1, p.err)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const int seen = limit - j * kBK;  // columns i < seen are visible
        uint32_t x[kBK / 32][32];
        __syncwarp();
#pragma unroll
        for (int c = 0; c < kBK / 32; ++c) tmem_ld_32_begin(s_tmem + c * 32, x[c]);
        // ---- the tile's maximum ----
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < kBK / 32; ++c) {
          tmem_ld_done(x[c]);
          if (c == 0) {  // (it waits for all of them) the next product may take the scores' place
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars[Smem::kSFree]);
          }
          if (seen < (c + 1) * 32) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (c * 32 + i >= seen) x[c][i] = 0xff800000u;  // -inf
          }
#pragma unroll
          for (int i = 0; i < 32; i += 2)
            m4[(i >> 1) & 3] = fmaxf(fmaxf(m4[(i >> 1) & 3], __uint_as_float(x[c][i])), __uint_as_float(x[c][i + 1]));
        }
        // (the scale is positive, so the largest score is the largest scaled one)
        const float top = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * p.scale_log2;
        const float m_new = fmaxf(m, top);
        // the product of the tile before has used its weights up, and O may be touched
        if (j > 0 && !mbar_wait_warp(&bars[Smem::kPvDone + x_tile], (g - 1) & 1, p.err)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const bool up = m_new > m + kRescaleLog2;  // also true for the first finite maximum
        if (__any_sync(0xffffffffu, up)) {
          const float alpha = up ? hw_exp2(m - m_new) : 1.f;
          if (up) m = m_new;
          l *= alpha;
          if (j > 0) {
#pragma unroll
            for (int c = 0; c < kV / 16; ++c) {
              uint32_t v[16];
              __syncwarp();
              tmem_ld_16(o_tmem + c * 16, v);
#pragma unroll
              for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
              tmem_st_16(o_tmem + c * 16, v);
            }
          }
        }
        // ---- the weights ----
        const float m_use = m == -INFINITY ? 0.f : m - kBias<T>;
        const uint64_t scale2 = pack2f(p.scale_log2, p.scale_log2), minus_m = pack2f(-m_use, -m_use);
        uint64_t l2[2] = {0, 0};
#pragma unroll
        for (int c = 0; c < kBK / 32; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint64_t y = fma2(pack2f(__uint_as_float(x[c][2 * i]), __uint_as_float(x[c][2 * i + 1])), scale2, minus_m);
            float e0, e1;
            unpack2f(y, e0, e1);
            e0 = hw_exp2(e0);
            e1 = hw_exp2(e1);
            l2[i & 1] = add2(l2[i & 1], pack2f(e0, e1));
            Pair<T>::store(reinterpret_cast<T*>(&pk[i]), e0, e1);
          }
          tmem_st_16(p_tmem + c * 16, pk);
        }
        {
          float a, b;
          unpack2f(add2(l2[0], l2[1]), a, b);
          l += a + b;
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[Smem::kPFull + x_tile]);
      }
      if (!ok) break;
      const int2 row = *row_of;
      T* const orow = static_cast<T*>(p.out) + int64_t(row.x) * p.o_tok + int64_t(row.y) * p.o_head;
      float* const lse = p.lse == nullptr || row.x < 0 ? nullptr : p.lse + int64_t(row.x) * p.lse_tok + row.y;
      if (tiles == 0) {  // no visible key: zero rows, as for an empty softmax
        if (row.x >= 0) {
#pragma unroll
          for (int c = 0; c < kV / 8; ++c) reinterpret_cast<uint4*>(orow)[c] = make_uint4(0u, 0u, 0u, 0u);
        }
        if (lse != nullptr) *lse = -INFINITY;
        continue;
      }
      // the item's last product is complete: O is final
      ok = mbar_wait_warp(&bars[Smem::kPvDone + x_tile], (g - 1) & 1, p.err);
      if (!ok) break;
      tc_fence_after();
      const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
      for (int c = 0; c < kV / 32; ++c) {
        uint32_t v[32];
        __syncwarp();
        tmem_ld_32(o_tmem + c * 32, v);
        if (row.x >= 0) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = l == 0.f ? 0.f : __uint_as_float(v[i * 8 + e]) * inv;
            *reinterpret_cast<Vec<T, 8>*>(orow + c * 32 + i * 8) = pack_f<T, 8>(f);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[Smem::kOFree + x_tile]);  // the next item may overwrite O
      if (lse != nullptr) *lse = l == 0.f ? -INFINITY : (m - kBias<T> + log2f(l)) * 0.6931471805599453f;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kAllocWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

// rows [tokens, heads, dim] (or [tokens, dim], heads 0): box = 128 tokens x one head x 64 columns
int make_rows_map(CUtensorMap* map, const void* base, bool bf16, int64_t dim, int64_t tokens, int64_t heads,
                  int64_t tok_stride, int64_t head_stride) {
  EncodeTiledFn enc = encode_fn();
  if (enc == nullptr) return fail(NTB200_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const cuuint64_t tok = cuuint64_t((tokens > 1 ? tok_stride : dim) * 2);
  const cuuint64_t dims3[3] = {cuuint64_t(dim), cuuint64_t(heads), cuuint64_t(tokens)};
  const cuuint64_t strides3[2] = {cuuint64_t((heads > 1 ? head_stride : dim) * 2), tok};
  const cuuint32_t box3[3] = {64, 1, 128};
  const cuuint64_t dims2[2] = {cuuint64_t(dim), cuuint64_t(tokens)};
  const cuuint64_t strides2[1] = {tok};
  const cuuint32_t box2[2] = {64, 128};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                         heads > 0 ? 3 : 2, const_cast<void*>(base), heads > 0 ? dims3 : dims2,
                         heads > 0 ? strides3 : strides2, heads > 0 ? box3 : box2, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(NTB200_ERR_CUDA, "cuTensorMapEncodeTiled (latent prefill) failed (%d)", int(r));
  return NTB200_OK;
}

template <typename T>
int launch_prefill(const CUtensorMap& q, const CUtensorMap& kn, const CUtensorMap& kr, const CUtensorMap& v,
                   const PrefillParams& p, int64_t ctas, int slot, cudaStream_t s) {
  const int st = ensure_smem_attribute(reinterpret_cast<const void*>(latent_prefill_kernel<T>), Smem::kBytes, slot);
  if (st != NTB200_OK) return st;
  return launch_kernel("latent_attention_prefill", latent_prefill_kernel<T>, dim3(unsigned(ctas)), dim3(kThreads),
                       Smem::kBytes, s, q, kn, kr, v, p);
}

}  // namespace
}  // namespace ntb200

extern "C" int ntb200_latent_attention_prefill(
    void* out, float* lse, const void* query, const void* k_nope, const void* k_rope, const void* value,
    const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int64_t num_seqs, int64_t num_q_tokens,
    int64_t num_k_tokens, int64_t num_heads, int64_t nope_dim, int64_t rope_dim, int64_t v_dim, int64_t max_query_len,
    float scale, int causal, int64_t q_token_stride, int64_t q_head_stride, int64_t kn_token_stride,
    int64_t kn_head_stride, int64_t kr_token_stride, int64_t v_token_stride, int64_t v_head_stride,
    int64_t out_token_stride, int64_t out_head_stride, int64_t lse_token_stride, int dtype, void* stream) {
  using namespace ntb200;
  if (dtype != NTB200_DTYPE_BF16 && dtype != NTB200_DTYPE_F16)
    return fail(NTB200_ERR_UNSUPPORTED_DTYPE, "latent_attention_prefill: dtype %d (bf16/f16 only)", dtype);
  if (nope_dim != kNope || rope_dim != kRope || v_dim != kV)
    return fail(NTB200_ERR_UNSUPPORTED_SHAPE,
                "latent_attention_prefill: nope_dim %lld / rope_dim %lld / v_dim %lld (128 / 64 / 128 only)",
                (long long)nope_dim, (long long)rope_dim, (long long)v_dim);
  if (num_seqs < 0 || num_q_tokens < 0 || num_k_tokens < 0 || num_heads <= 0 || max_query_len < 0)
    return fail(NTB200_ERR_INVALID_ARGUMENT, "latent_attention_prefill: bad sizes");
  if (!(scale > 0.f))
    return fail(NTB200_ERR_INVALID_ARGUMENT, "latent_attention_prefill: scale must be positive");
  if (num_seqs == 0 || num_q_tokens == 0 || max_query_len == 0) return NTB200_OK;
  constexpr int64_t kMost = 0x7fffffff - 1024;  // row numbers rounded up to a tile stay 32-bit
  if (num_heads > 65535 || num_q_tokens > kMost || num_k_tokens > kMost || num_seqs > kMost ||
      ceil_div(num_q_tokens, kItemRows) + num_seqs > kMost / num_heads)
    return fail(NTB200_ERR_UNSUPPORTED_SHAPE, "latent_attention_prefill: sizes beyond the launch limits");
  if (!out || !query || !cu_seqlens_q || !cu_seqlens_k || (num_k_tokens > 0 && (!k_nope || !k_rope || !value)))
    return fail(NTB200_ERR_INVALID_ARGUMENT, "latent_attention_prefill: null pointer");
  if (!aligned16(out) || !aligned16(query) || !aligned16(k_nope) || !aligned16(k_rope) || !aligned16(value) ||
      q_token_stride % 8 || q_head_stride % 8 || kn_token_stride % 8 || kn_head_stride % 8 || kr_token_stride % 8 ||
      v_token_stride % 8 || v_head_stride % 8 || out_token_stride % 8 || out_head_stride % 8)
    return fail(NTB200_ERR_MISALIGNED, "latent_attention_prefill: pointers 16-byte aligned, strides multiples of 8");
  const bool bf16 = dtype == NTB200_DTYPE_BF16;
  CUtensorMap q, kn, kr, v;
  int st = make_rows_map(&q, query, bf16, kNope + kRope, num_q_tokens, num_heads, q_token_stride, q_head_stride);
  if (st != NTB200_OK) return st;
  kn = kr = v = q;  // never read when there are no keys
  if (num_k_tokens > 0) {
    st = make_rows_map(&kn, k_nope, bf16, kNope, num_k_tokens, num_heads, kn_token_stride, kn_head_stride);
    if (st == NTB200_OK) st = make_rows_map(&kr, k_rope, bf16, kRope, num_k_tokens, 0, kr_token_stride, 0);
    if (st == NTB200_OK) st = make_rows_map(&v, value, bf16, kV, num_k_tokens, num_heads, v_token_stride, v_head_stride);
    if (st != NTB200_OK) return st;
  }
  PrefillParams p = {};
  p.out = out;
  p.lse = lse;
  p.cu_q = cu_seqlens_q;
  p.cu_k = cu_seqlens_k;
  p.o_tok = out_token_stride;
  p.o_head = out_head_stride;
  p.lse_tok = lse_token_stride;
  p.num_seqs = int(num_seqs);
  p.num_q = int(num_q_tokens);
  p.num_k = int(num_k_tokens);
  p.num_heads = int(num_heads);
  p.causal = causal != 0;
  p.scale_log2 = scale * 1.4426950408889634f;  // softmax in the exp2 domain
  p.err = device_error_word();
  // no more CTAs than there can be items: every sequence rounds up at most once
  const int64_t by_len = ceil_div(std::min(max_query_len, num_q_tokens), kItemRows) * num_seqs;
  const int64_t by_tokens = ceil_div(num_q_tokens, kItemRows) + num_seqs;
  const int64_t ctas = std::min<int64_t>(std::min(by_len, by_tokens) * num_heads, num_sms());
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return bf16 ? launch_prefill<__nv_bfloat16>(q, kn, kr, v, p, ctas, 134, s)
              : launch_prefill<__half>(q, kn, kr, v, p, ctas, 135, s);
}
