// One latent-attention layer's rows on their way into the paged cache, in one launch:
//   latent[t]  -> y = latent[t] * rsqrt(mean(latent[t]^2) + eps) * weight   (or unchanged)
//   key[t]     -> rotated in place (the one rotary key of the token, shared by all heads)
//   query[t,h] -> rotated in place (the rotary part of every head)
//   cache[slot_mapping[t]] = [y | rotated key[t]]
// Statistics, products and rotations are fp32; y and the rotated values are rounded once.
//
// Warps take units: unit 0 of a token is its latent row and key (one warp holds the row in
// registers, so it is read once and no barrier is needed), the others are a few vectors a lane
// of its query heads.  HBM-bound for prefill batches, one launch's latency for decode.
#include "common.cuh"
#include "rope_layout.cuh"

namespace ntb200 {
namespace {

constexpr int kThreads = 256;
constexpr int kVec = 8;                       // 16 bytes of a 16-bit type
constexpr int kMaxLatent = 1024;              // a lane holds latent_dim / 256 vectors
constexpr int kLatentVecs = kMaxLatent / (32 * kVec);
constexpr int kMaxRope = 256;

struct StoreParams {
  const void* positions;
  int positions_i64;
  const void* slots;
  int slots_i64;
  int64_t num_tokens, num_store;
  int num_heads, latent_dim, rope_dim;
  int64_t q_tok, q_head, lat_tok, key_tok, lat_out_tok;
  int64_t table_row, table_rows;
  int64_t block_size, num_slots, block_stride, page_stride;
  float eps;
  unsigned int* err;
};

template <typename T, typename C, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads)
    latent_store_kernel(T* __restrict__ q, const T* latent, T* __restrict__ key, const T* __restrict__ weight,
                        const C* __restrict__ table, T* __restrict__ cache, T* latent_out, const StoreParams p) {
  const int lane = threadIdx.x & 31;
  constexpr int kUnit = 32 * kRotItems;
  const int q_vecs = p.num_heads * rot_vectors<kVec, INTERLEAVED>(p.rope_dim);
  const int units = 1 + (q_vecs + kUnit - 1) / kUnit;
  const int64_t u = int64_t(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  pdl_trigger();
  pdl_wait();
  if (u >= p.num_tokens * units) return;
  const int64_t t = u / units;
  const int unit = int(u - t * units);
  const auto row = [&]() -> const C* {
    const int64_t pos = p.positions_i64 ? static_cast<const int64_t*>(p.positions)[t]
                                        : static_cast<const int32_t*>(p.positions)[t];
    if (pos < 0 || pos >= p.table_rows) {  // not rotated; flagged once
      if (unit == 0 && lane == 0) raise_device_error(p.err, NTB200_DEVERR_INDEX_RANGE);
      return nullptr;
    }
    return table + pos * p.table_row;
  };
  if (unit > 0) {
    const TokenHeads<T> heads = {q + t * p.q_tok, nullptr, p.num_heads, 0, p.q_head, 0};
    rotate_unit<T, C, kVec, INTERLEAVED, kRotItems>(heads, (unit - 1) * kUnit, p.rope_dim, row);
    return;
  }

  // ---- the latent row and the key ----
  const int vecs = p.latent_dim / kVec;
  float x[kLatentVecs][kVec];
#pragma unroll
  for (int j = 0; j < kLatentVecs; ++j)
    if (lane + 32 * j < vecs) load_f<T, kVec>(latent + t * p.lat_tok + (lane + 32 * j) * kVec, x[j]);
  int64_t slot = -1;
  if (t < p.num_store) {
    slot = p.slots_i64 ? static_cast<const int64_t*>(p.slots)[t] : static_cast<const int32_t*>(p.slots)[t];
    if (slot >= p.num_slots) {
      if (lane == 0) raise_device_error(p.err, NTB200_DEVERR_INDEX_RANGE);
      slot = -1;
    }
  }
  T* const dst = cache + (slot >= 0 ? slot / p.block_size * p.block_stride + slot % p.block_size * p.page_stride : 0);
  // the key: lanes 0.. hold its vectors
  using Item = RotItem<T, kVec, INTERLEAVED>;
  const int key_vecs = rot_vectors<kVec, INTERLEAVED>(p.rope_dim);
  const int half = p.rope_dim / 2;
  if (lane < key_vecs) {
    Item item;
    T* const at = key + t * p.key_tok + lane * kVec;
    item.load(at, half);
    if (const C* cs = row()) {
      float c[Item::kPairs], s[Item::kPairs];
      const int o = INTERLEAVED ? lane * kVec / 2 : lane * kVec;
      load_table<C, Item::kPairs>(cs + o, c);
      load_table<C, Item::kPairs>(cs + half + o, s);
      item.rotate(c, s);
      item.store(at, half);
    }
    if (slot >= 0) item.store(dst + p.latent_dim + lane * kVec, half);
  }
  float inv = 1.f;
  if (weight != nullptr) {
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < kLatentVecs; ++j)
      if (lane + 32 * j < vecs)
#pragma unroll
        for (int e = 0; e < kVec; ++e) sum += x[j][e] * x[j][e];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    inv = rsqrtf(sum / float(p.latent_dim) + p.eps);
  }
#pragma unroll
  for (int j = 0; j < kLatentVecs; ++j) {
    const int v = lane + 32 * j;
    if (v >= vecs) continue;
    if (weight != nullptr) {
      float w[kVec];
      load_f<T, kVec>(weight + v * kVec, w);
#pragma unroll
      for (int e = 0; e < kVec; ++e) x[j][e] = x[j][e] * inv * w[e];
    }
    const Vec<T, kVec> y = pack_f<T, kVec>(x[j]);
    if (slot >= 0) *reinterpret_cast<Vec<T, kVec>*>(dst + v * kVec) = y;
    if (latent_out != nullptr) *reinterpret_cast<Vec<T, kVec>*>(latent_out + t * p.lat_out_tok + v * kVec) = y;
  }
}

template <typename T, typename C, bool INTERLEAVED>
int launch_store(void* q, const void* latent, void* key, const void* weight, const void* table, void* cache,
                 void* latent_out, const StoreParams& p, cudaStream_t stream) {
  const int64_t units = 1 + ceil_div(int64_t(p.num_heads) * rot_vectors<kVec, INTERLEAVED>(p.rope_dim), 32 * kRotItems);
  const int64_t ctas = ceil_div(p.num_tokens * units, kThreads / 32);
  if (ctas > 0x7fffffff) return fail(NTB200_ERR_UNSUPPORTED_SHAPE, "latent_rope_and_cache: too many tokens");
  return launch_kernel("latent_rope_and_cache", latent_store_kernel<T, C, INTERLEAVED>, dim3(unsigned(ctas)),
                       dim3(kThreads), 0, stream, static_cast<T*>(q), static_cast<const T*>(latent),
                       static_cast<T*>(key), static_cast<const T*>(weight), static_cast<const C*>(table),
                       static_cast<T*>(cache), static_cast<T*>(latent_out), p);
}

template <typename T>
int by_form(bool f32_table, bool interleaved, void* q, const void* latent, void* key, const void* weight,
            const void* table, void* cache, void* latent_out, const StoreParams& p, cudaStream_t s) {
  if (f32_table)
    return interleaved ? launch_store<T, float, true>(q, latent, key, weight, table, cache, latent_out, p, s)
                       : launch_store<T, float, false>(q, latent, key, weight, table, cache, latent_out, p, s);
  return interleaved ? launch_store<T, T, true>(q, latent, key, weight, table, cache, latent_out, p, s)
                     : launch_store<T, T, false>(q, latent, key, weight, table, cache, latent_out, p, s);
}

}  // namespace
}  // namespace ntb200

extern "C" int ntb200_latent_rope_and_cache(
    const void* positions, int positions_dtype, void* query, const void* latent, void* key, const void* norm_weight,
    float eps, const void* cos_sin_cache, int cache_dtype, int interleaved, void* kv_cache, void* latent_out,
    const void* slot_mapping, int slot_dtype, int64_t num_tokens, int64_t num_store_tokens, int64_t num_heads,
    int64_t latent_dim, int64_t rope_dim, int64_t q_token_stride, int64_t q_head_stride, int64_t latent_token_stride,
    int64_t key_token_stride, int64_t latent_out_token_stride, int64_t cos_sin_row_stride, int64_t num_cos_sin_rows,
    int64_t block_size, int64_t num_slots, int64_t cache_block_stride, int64_t cache_page_stride, int dtype,
    void* stream) {
  using namespace ntb200;
  if (dtype != NTB200_DTYPE_BF16 && dtype != NTB200_DTYPE_F16)
    return fail(NTB200_ERR_UNSUPPORTED_DTYPE, "latent_rope_and_cache: dtype %d (bf16/f16 only)", dtype);
  if (cache_dtype != dtype && cache_dtype != NTB200_DTYPE_F32)
    return fail(NTB200_ERR_UNSUPPORTED_DTYPE, "latent_rope_and_cache: cos_sin_cache dtype %d (query's or fp32)", cache_dtype);
  if ((positions_dtype != NTB200_DTYPE_I64 && positions_dtype != NTB200_DTYPE_I32) ||
      (slot_dtype != NTB200_DTYPE_I64 && slot_dtype != NTB200_DTYPE_I32))
    return fail(NTB200_ERR_UNSUPPORTED_DTYPE, "latent_rope_and_cache: positions and slots must be int32 or int64");
  if (num_tokens < 0 || num_store_tokens < 0 || num_store_tokens > num_tokens || num_heads < 0 || block_size <= 0 ||
      num_slots < 0 || num_cos_sin_rows < 0)
    return fail(NTB200_ERR_INVALID_ARGUMENT, "latent_rope_and_cache: bad sizes");
  if (latent_dim <= 0 || latent_dim > kMaxLatent || latent_dim % kVec != 0 || rope_dim <= 0 || rope_dim > kMaxRope ||
      rope_dim % 16 != 0 || num_heads > 0x7fffffff / kMaxRope)
    return fail(NTB200_ERR_UNSUPPORTED_SHAPE,
                "latent_rope_and_cache: latent_dim %lld (a multiple of 8 up to 1024), rope_dim %lld (of 16 up to 256)",
                (long long)latent_dim, (long long)rope_dim);
  if (cos_sin_row_stride < rope_dim || latent_token_stride < (num_tokens > 1 ? latent_dim : 0) ||
      key_token_stride < (num_tokens > 1 ? rope_dim : 0) || cache_page_stride < latent_dim + rope_dim)
    return fail(NTB200_ERR_INVALID_ARGUMENT, "latent_rope_and_cache: a row stride is below its row");
  if (num_tokens == 0) return NTB200_OK;
  if (query == nullptr) num_heads = 0;
  if (!positions || !latent || !key || !cos_sin_cache || !kv_cache || (!slot_mapping && num_store_tokens > 0))
    return fail(NTB200_ERR_INVALID_ARGUMENT, "latent_rope_and_cache: null pointer");
  const int64_t table_step = 16 / dtype_size(cache_dtype);
  if (!aligned16(query) || !aligned16(latent) || !aligned16(key) || !aligned16(norm_weight) || !aligned16(kv_cache) ||
      !aligned16(latent_out) || !aligned16(cos_sin_cache) || q_token_stride % 8 || q_head_stride % 8 ||
      latent_token_stride % 8 || key_token_stride % 8 || latent_out_token_stride % 8 || cache_block_stride % 8 ||
      cache_page_stride % 8 || cos_sin_row_stride % table_step || (rope_dim / 2) % table_step)
    return fail(NTB200_ERR_MISALIGNED, "latent_rope_and_cache: pointers 16-byte aligned, strides multiples of 8");
  StoreParams p = {};
  p.positions = positions;
  p.positions_i64 = positions_dtype == NTB200_DTYPE_I64;
  p.slots = slot_mapping;
  p.slots_i64 = slot_dtype == NTB200_DTYPE_I64;
  p.num_tokens = num_tokens;
  p.num_store = num_store_tokens;
  p.num_heads = int(num_heads);
  p.latent_dim = int(latent_dim);
  p.rope_dim = int(rope_dim);
  p.q_tok = q_token_stride;
  p.q_head = q_head_stride;
  p.lat_tok = latent_token_stride;
  p.key_tok = key_token_stride;
  p.lat_out_tok = latent_out_token_stride;
  p.table_row = cos_sin_row_stride;
  p.table_rows = num_cos_sin_rows;
  p.block_size = block_size;
  p.num_slots = num_slots;
  p.block_stride = cache_block_stride;
  p.page_stride = cache_page_stride;
  p.eps = eps;
  p.err = device_error_word();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool f32 = cache_dtype == NTB200_DTYPE_F32, inter = interleaved != 0;
  return dtype == NTB200_DTYPE_BF16
             ? by_form<__nv_bfloat16>(f32, inter, query, latent, key, norm_weight, cos_sin_cache, kv_cache, latent_out, p, s)
             : by_form<__half>(f32, inter, query, latent, key, norm_weight, cos_sin_cache, kv_cache, latent_out, p, s);
}
