// Rotary positions in both layouts, and the cos/sin table of long contexts.
//
// rotary_embedding: in place on the first rotary_dim elements of every query and key head,
// read and written once; a warp takes a few vectors a lane of one token's heads, so that one
// decode token spreads over many warps.  Bound by HBM.
//
// rope_cos_sin_cache: row p holds cos(p f_i) and sin(p f_i) of every frequency f_i.  An fp32
// product p * f_i is off by up to 2^-24 of the angle, 0.008 rad at 128 Ki positions and more
// beyond: a CTA forms its frequencies once in fp64, in turns, and its threads walk rows with them in
// 64-bit fixed point, where an angle is one addition (off by 2^-64 turns a row, on top of the
// frequency's error, at most (7 ln(base) + 13) 2^-53 of the angle: ln(base), its product with i, exp, the
// scaling and 1 / (2 pi) each round, the first ones in an exponent of up to ln(base)); only what is left
// beside the nearest quarter turn goes to fp32
// (off by at most 2^-23 rad).  131075 rows of 32 frequencies in fp32: 7.5 us, 4.5 TB/s of stores
// (11.7 with the library's sine and cosine, 86 instructions an angle, and a frequency a thread).
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "rope_layout.cuh"

namespace ntb200 {
namespace {

constexpr int kThreads = 256;

template <typename T, typename C, int VEC, bool INTERLEAVED, int ITEMS, typename P>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const P* __restrict__ positions, T* __restrict__ q,
                                                          T* __restrict__ k, const C* __restrict__ table,
                                                          int64_t num_tokens, int num_q, int num_k, int rot,
                                                          int64_t q_tok, int64_t q_head, int64_t k_tok, int64_t k_head,
                                                          int64_t table_row, int64_t table_rows, unsigned int* err) {
  constexpr int kUnit = 32 * ITEMS;
  const int total = (num_q + num_k) * rot_vectors<VEC, INTERLEAVED>(rot);
  const int units = (total + kUnit - 1) / kUnit;
  const int64_t u = int64_t(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  pdl_trigger();
  pdl_wait();
  if (u >= num_tokens * units) return;
  const int64_t t = u / units;
  const int first = int(u - t * units) * kUnit;
  const TokenHeads<T> heads = {q + t * q_tok, k + t * k_tok, num_q, num_k, q_head, k_head};
  rotate_unit<T, C, VEC, INTERLEAVED, ITEMS>(heads, first, rot, [&]() -> const C* {
    const int64_t pos = static_cast<int64_t>(positions[t]);
    if (pos < 0 || pos >= table_rows) {  // the token stays untouched; flagged once
      if (first == 0 && (threadIdx.x & 31) == 0) raise_device_error(err, NTB200_DEVERR_INDEX_RANGE);
      return nullptr;
    }
    return table + pos * table_row;
  });
}

struct RotaryCall {
  const void* positions;
  int positions_dtype;
  void *q, *k;
  const void* table;
  int64_t tokens, hq, hk, rot, qt, qh, kt, kh, row, rows;
  cudaStream_t stream;
};

template <typename T, typename C, int VEC, bool INTERLEAVED, int ITEMS, typename P>
int launch_items(const RotaryCall& c, int64_t total) {
  const int64_t units = c.tokens * ceil_div(total, 32 * ITEMS);
  const int64_t ctas = ceil_div(units, kThreads / 32);
  if (ctas > 0x7fffffff) return fail(NTB200_ERR_UNSUPPORTED_SHAPE, "rotary_embedding: too many tokens");
  return launch_kernel("rotary_embedding", rotary_kernel<T, C, VEC, INTERLEAVED, ITEMS, P>, dim3(unsigned(ctas)),
                       dim3(kThreads), 0, c.stream, static_cast<const P*>(c.positions), static_cast<T*>(c.q),
                       static_cast<T*>(c.k), static_cast<const C*>(c.table), c.tokens, int(c.hq), int(c.hk),
                       int(c.rot), c.qt, c.qh, c.kt, c.kh, c.row, c.rows, device_error_word());
}

template <typename T, typename C, int VEC, bool INTERLEAVED, typename P>
int launch_rotary(const RotaryCall& c) {
  const int64_t total = (c.hq + c.hk) * rot_vectors<VEC, INTERLEAVED>(int(c.rot));
  if (total == 0) return NTB200_OK;
  // a call that leaves SMs idle is spread one vector a lane (7 tokens of 40 heads: 1.8 us against 2.2)
  if (c.tokens * ceil_div(total, 32 * kRotItems) < int64_t(num_sms()) * 8)
    return launch_items<T, C, VEC, INTERLEAVED, 1, P>(c, total);
  return launch_items<T, C, VEC, INTERLEAVED, kRotItems, P>(c, total);
}

template <typename T, typename C, int VEC, bool INTERLEAVED>
int by_position(const RotaryCall& c) {
  return c.positions_dtype == NTB200_DTYPE_I64 ? launch_rotary<T, C, VEC, INTERLEAVED, int64_t>(c)
                                               : launch_rotary<T, C, VEC, INTERLEAVED, int32_t>(c);
}

template <typename T, typename C>
int by_layout(const RotaryCall& c, bool interleaved) {
  constexpr int kVec = 16 / sizeof(T);
  const int64_t half = c.rot / 2;
  // 16-byte vectors need aligned bases and strides, whole vectors a head (or head half), and
  // table halves that start on 16 bytes; anything else goes pair by pair
  const bool vec = aligned16(c.q) && c.qt % kVec == 0 && c.qh % kVec == 0 &&
                   (c.hk == 0 || (aligned16(c.k) && c.kt % kVec == 0 && c.kh % kVec == 0)) &&
                   (interleaved ? c.rot : half) % kVec == 0 && aligned16(c.table) &&
                   (c.row * sizeof(C)) % 16 == 0 && (half * sizeof(C)) % 16 == 0;
  if (interleaved) {
    // a lone pair is one access of two elements: it needs their alignment
    const bool pair = reinterpret_cast<uintptr_t>(c.q) % (2 * sizeof(T)) == 0 && c.qt % 2 == 0 && c.qh % 2 == 0 &&
                      (c.hk == 0 ||
                       (reinterpret_cast<uintptr_t>(c.k) % (2 * sizeof(T)) == 0 && c.kt % 2 == 0 && c.kh % 2 == 0));
    if (vec) return by_position<T, C, kVec, true>(c);
    if (!pair) return fail(NTB200_ERR_MISALIGNED, "rotary_embedding: interleaved pairs must be aligned to their size");
    return by_position<T, C, 2, true>(c);
  }
  return vec ? by_position<T, C, kVec, false>(c) : by_position<T, C, 1, false>(c);
}

template <typename T>
int by_table(const RotaryCall& c, int table_dtype, int dtype, bool interleaved) {
  if (table_dtype == dtype) return by_layout<T, T>(c, interleaved);
  return by_layout<T, float>(c, interleaved);
}

// ---- the table ----

struct TableParams {
  int64_t rows, first, row_stride;
  int half;
  int thread_rows;    // rows a thread forms
  double log_step;    // ln f_{i+1} - ln f_i before scaling
  double linear;      // every frequency times this (1: unscaled)
  double ramp_lo, ramp_inv;  // yarn: share of the divided frequency = clamp((i - lo) * inv, 0, 1)
  double yarn;        // 1 / factor of the divided frequency; 0: no yarn
  float magnitude;
  const float* divisors;
};

// cos and sin, each times `mag`, of two angles in units of 2^-64 turns.  The nearest quarter turn is
// the top two bits (rounded) and costs nothing; the rest, y with |y| <= pi / 4, takes the Taylor
// series up to y^9 and y^10, whose next terms are below 2e-9 and 2e-10.  Both angles go through
// one instruction stream (f32x2).
__device__ __forceinline__ void cos_sin_2(uint64_t a, uint64_t b, uint64_t mag, float (&c)[2], float (&s)[2]) {
  constexpr float kStep = float(1.5707963267948966 / 4294967296.0);  // 2^-32 quarter turns in radians
  const auto both = [](double v) { return pack2f(float(v), float(v)); };
  const float ya = float(static_cast<int32_t>((a << 2) >> 32)), yb = float(static_cast<int32_t>((b << 2) >> 32));
  const uint64_t y = mul2(pack2f(ya, yb), pack2f(kStep, kStep));
  const uint64_t z = mul2(y, y);
  uint64_t p = fma2(z, both(1.0 / 362880), both(-1.0 / 5040));
  p = fma2(p, z, both(1.0 / 120));
  p = fma2(p, z, both(-1.0 / 6));
  const uint64_t sn = mul2(fma2(mul2(y, z), p, y), mag);
  p = fma2(z, both(-1.0 / 3628800), both(1.0 / 40320));
  p = fma2(p, z, both(-1.0 / 720));
  p = fma2(p, z, both(1.0 / 24));
  p = fma2(p, z, both(-0.5));
  const uint64_t cn = mul2(fma2(p, z, both(1.0)), mag);
  float sv[2], cv[2];
  unpack2f(sn, sv[0], sv[1]);
  unpack2f(cn, cv[0], cv[1]);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t q = (static_cast<uint32_t>((i == 0 ? a : b) >> 32) + 0x20000000u) >> 30;
    const float u = (q & 1) ? cv[i] : sv[i], v = (q & 1) ? sv[i] : cv[i];
    s[i] = __uint_as_float(__float_as_uint(u) ^ ((q & 2) << 30));
    c[i] = __uint_as_float(__float_as_uint(v) ^ (((q + 1) & 2) << 30));
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) cos_sin_kernel(T* __restrict__ out, const TableParams p) {
  pdl_trigger();
  pdl_wait();
  const int lanes = p.half < kThreads ? p.half : kThreads;  // threads along the frequencies
  const int strip = kThreads / lanes;                       // rows a CTA writes at once
  struct Frequency {
    uint64_t unit;  // its part of a turn in units of 2^-64 turns
    float mag;      // of its cosines and sines
  };
  const auto frequency = [&](int i) -> Frequency {
    double f = exp(i * p.log_step) * p.linear;
    if (p.yarn != 0.0) {
      const double share = fmin(fmax((i - p.ramp_lo) * p.ramp_inv, 0.0), 1.0);
      f = f * p.yarn * share + f * (1.0 - share);
    }
    if (p.divisors != nullptr) f /= double(p.divisors[i]);
    // whole turns count for nothing: the angle of a row is its number times f's part of a turn, whose
    // 64-bit product and sums drop the whole turns by themselves
    f *= 0.15915494309189535;
    // a divisor of 0 or NaN leaves no frequency, and an integer cannot say so: the magnitude does
    if (!isfinite(f)) return {0, __int_as_float(0x7fffffff)};
    return {static_cast<uint64_t>((f - floor(f)) * 18446744073709551616.0), p.magnitude};
  };
  __shared__ Frequency shared[kThreads / 2];  // where several threads need a frequency one forms it
  if (strip > 1) {
    if (int(threadIdx.x) < lanes) shared[threadIdx.x] = frequency(threadIdx.x);
    __syncthreads();
  }
  if (int(threadIdx.x) >= strip * lanes) return;
  const int64_t row0 = int64_t(blockIdx.x) * strip * p.thread_rows + threadIdx.x / lanes;
  for (int i = threadIdx.x % lanes; i < p.half; i += lanes) {
    const Frequency own = strip > 1 ? shared[i] : frequency(i);
    const uint64_t unit = own.unit;
    const uint64_t step = unit * static_cast<uint64_t>(strip);
    uint64_t phase = unit * static_cast<uint64_t>(p.first + row0);
    const uint64_t mag = pack2f(own.mag, own.mag);
    const int64_t left = p.rows - row0;  // (this thread's rows are strip apart)
    const int n = int(left <= 0 ? 0 : min((left + strip - 1) / strip, int64_t(p.thread_rows)));
    const int64_t ahead = strip * p.row_stride;
    T* o = out + row0 * p.row_stride + i;
#pragma unroll 2
    for (int r = 0; r < n; r += 2, phase += 2 * step, o += 2 * ahead) {
      float s[2], c[2];
      cos_sin_2(phase, phase + step, mag, c, s);
      o[0] = Elem<T>::from_f(c[0]);
      o[p.half] = Elem<T>::from_f(s[0]);
      if (r + 1 < n) {
        o[ahead] = Elem<T>::from_f(c[1]);
        o[ahead + p.half] = Elem<T>::from_f(s[1]);
      }
    }
  }
}

// Rows a thread: as many as make one wave of four CTAs an SM (131075 x 64, measured side by side: 7.2 us with four, 8.0 with
// five, 8.6 with two or three; 8.4 in waves of 16 rows a thread).
template <typename T>
int launch_table(void* out, TableParams p, cudaStream_t stream) {
  const int lanes = p.half < kThreads ? p.half : kThreads;
  const int strip = kThreads / lanes;
  const int64_t per = ceil_div(p.rows, int64_t(strip) * num_sms() * 4);
  p.thread_rows = int(std::min<int64_t>(std::max<int64_t>(per, 2), 1 << 30));
  const int64_t ctas = ceil_div(p.rows, int64_t(strip) * p.thread_rows);
  if (ctas > 0x7fffffff) return fail(NTB200_ERR_UNSUPPORTED_SHAPE, "rope_cos_sin_cache: too many rows");
  return launch_kernel("rope_cos_sin_cache", cos_sin_kernel<T>, dim3(unsigned(ctas)), dim3(kThreads), 0, stream,
                       static_cast<T*>(out), p);
}

}  // namespace
}  // namespace ntb200

extern "C" int ntb200_rotary_embedding(const void* positions, int positions_dtype, void* query, void* key,
                                       const void* cos_sin_cache, int cache_dtype, int64_t num_tokens,
                                       int64_t num_q_heads, int64_t num_k_heads, int64_t head_size, int64_t rotary_dim,
                                       int interleaved, int64_t q_token_stride, int64_t q_head_stride,
                                       int64_t k_token_stride, int64_t k_head_stride, int64_t cache_row_stride,
                                       int64_t num_cache_rows, int dtype, void* stream) {
  using namespace ntb200;
  if (dtype != NTB200_DTYPE_F32 && dtype != NTB200_DTYPE_BF16 && dtype != NTB200_DTYPE_F16)
    return fail(NTB200_ERR_UNSUPPORTED_DTYPE, "rotary_embedding: dtype %d", dtype);
  if (cache_dtype != dtype && cache_dtype != NTB200_DTYPE_F32)
    return fail(NTB200_ERR_UNSUPPORTED_DTYPE, "rotary_embedding: cos_sin_cache dtype %d (query's or fp32)", cache_dtype);
  if (positions_dtype != NTB200_DTYPE_I64 && positions_dtype != NTB200_DTYPE_I32)
    return fail(NTB200_ERR_UNSUPPORTED_DTYPE, "rotary_embedding: positions dtype %d", positions_dtype);
  if (num_tokens < 0 || num_q_heads < 0 || num_k_heads < 0 || head_size <= 0 || num_cache_rows < 0)
    return fail(NTB200_ERR_INVALID_ARGUMENT, "rotary_embedding: bad shape");
  if (rotary_dim <= 0 || rotary_dim > head_size || rotary_dim % 2 != 0)
    return fail(NTB200_ERR_INVALID_ARGUMENT, "rotary_embedding: rotary_dim must be even and <= head_size");
  if (cache_row_stride < rotary_dim)
    return fail(NTB200_ERR_INVALID_ARGUMENT, "rotary_embedding: cache row stride < rotary_dim");
  if (key == nullptr) num_k_heads = 0;
  if (num_tokens == 0 || num_q_heads + num_k_heads == 0) return NTB200_OK;
  if (positions == nullptr || (query == nullptr && num_q_heads > 0) || cos_sin_cache == nullptr)
    return fail(NTB200_ERR_INVALID_ARGUMENT, "rotary_embedding: null pointer");
  if (rotary_dim > 0x7fffffff || num_q_heads > 0x7fffffff || num_k_heads > 0x7fffffff ||
      (num_q_heads + num_k_heads) > 0x7fffffff / rotary_dim)
    return fail(NTB200_ERR_UNSUPPORTED_SHAPE, "rotary_embedding: too many heads");
  const RotaryCall c = {positions,      positions_dtype, query,          key,           cos_sin_cache,
                        num_tokens,     num_q_heads,     num_k_heads,    rotary_dim,    q_token_stride,
                        q_head_stride,  k_token_stride,  k_head_stride,  cache_row_stride,
                        num_cache_rows, static_cast<cudaStream_t>(stream)};
  const bool inter = interleaved != 0;
  if (dtype == NTB200_DTYPE_F32) return by_layout<float, float>(c, inter);
  if (dtype == NTB200_DTYPE_BF16) return by_table<__nv_bfloat16>(c, cache_dtype, dtype, inter);
  return by_table<__half>(c, cache_dtype, dtype, inter);
}

extern "C" int ntb200_rope_cos_sin_cache(void* out, int64_t num_positions, int64_t first_position, int64_t rotary_dim,
                                         double base, int scaling, double factor, double original_max_position,
                                         double beta_fast, double beta_slow, double magnitude,
                                         const float* freq_divisors, int64_t out_row_stride, int dtype, void* stream) {
  using namespace ntb200;
  if (dtype != NTB200_DTYPE_F32 && dtype != NTB200_DTYPE_BF16 && dtype != NTB200_DTYPE_F16)
    return fail(NTB200_ERR_UNSUPPORTED_DTYPE, "rope_cos_sin_cache: dtype %d", dtype);
  if (num_positions < 0 || first_position < 0 || rotary_dim <= 0 || rotary_dim % 2 != 0 || out_row_stride < rotary_dim)
    return fail(NTB200_ERR_INVALID_ARGUMENT, "rope_cos_sin_cache: bad shape");
  if (scaling < NTB200_ROPE_NONE || scaling > NTB200_ROPE_YARN)
    return fail(NTB200_ERR_INVALID_ARGUMENT, "rope_cos_sin_cache: unknown scaling %d", scaling);
  if (!(base > 1.0) || std::isinf(base) || !(factor > 0.0) || std::isinf(factor) || !std::isfinite(magnitude))
    return fail(NTB200_ERR_INVALID_ARGUMENT, "rope_cos_sin_cache: base must be over 1, factor over 0, all finite");
  if (scaling == NTB200_ROPE_YARN && (!(original_max_position > 0.0) || std::isinf(original_max_position) ||
                                      !(beta_slow > 0.0) || !(beta_fast >= beta_slow) || std::isinf(beta_fast)))
    return fail(NTB200_ERR_INVALID_ARGUMENT, "rope_cos_sin_cache: yarn needs an original length and beta_fast >= beta_slow > 0");
  if (rotary_dim > 65536 || first_position > (int64_t(1) << 40) || num_positions > (int64_t(1) << 40))
    return fail(NTB200_ERR_UNSUPPORTED_SHAPE, "rope_cos_sin_cache: sizes beyond the launch limits");
  if (num_positions == 0) return NTB200_OK;
  if (out == nullptr) return fail(NTB200_ERR_INVALID_ARGUMENT, "rope_cos_sin_cache: null pointer");
  const double d = double(rotary_dim);
  TableParams p = {};
  p.rows = num_positions;
  p.first = first_position;
  p.row_stride = out_row_stride;
  p.half = int(rotary_dim / 2);
  // ntk: the base grows so that the last frequency is divided by exactly `factor`
  const double ntk = scaling == NTB200_ROPE_NTK && rotary_dim > 2 ? std::log(factor) * d / (d - 2.0) : 0.0;
  p.log_step = -2.0 / d * (std::log(base) + ntk);
  p.linear = scaling == NTB200_ROPE_LINEAR ? 1.0 / factor : 1.0;
  if (scaling == NTB200_ROPE_YARN) {
    // frequency i makes original_max_position * f_i / (2 pi) turns over the trained length: those
    // with over beta_fast turns stay, those with under beta_slow are divided, a ramp between
    const double kTurn = 6.283185307179586;
    auto at = [&](double turns) { return d * std::log(original_max_position / (turns * kTurn)) / (2.0 * std::log(base)); };
    const double lo = std::fmax(std::floor(at(beta_fast)), 0.0);
    const double hi = std::fmin(std::ceil(at(beta_slow)), d - 1.0);
    p.yarn = 1.0 / factor;
    p.ramp_lo = lo;
    p.ramp_inv = 1.0 / std::fmax(hi - lo, 0.001);
  }
  p.magnitude = float(magnitude);
  p.divisors = freq_divisors;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == NTB200_DTYPE_F32) return launch_table<float>(out, p, s);
  if (dtype == NTB200_DTYPE_BF16) return launch_table<__nv_bfloat16>(out, p, s);
  return launch_table<__half>(out, p, s);
}
