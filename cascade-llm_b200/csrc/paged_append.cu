// Rotary positions of new tokens' q and k, with k and v written into the
// pages of their sequences in the same pass.
//
// Token n at position p, rotary frequency f_i, pair (a, b) of a head:
//   (a, b) -> c * (a cos(p f_i) - b sin(p f_i), b cos(p f_i) + a sin(p f_i)).
// The angle p * f_i has up to 55 bits and its whole turns tell nothing: it is formed
// as a double and the product's rounding error, and reduced to [-pi, pi] with 2 pi
// in two parts (Cody and Waite's reduction), then split into a 32-bit part and its
// remainder, which corrects sine and cosine to first order. A 32-bit angle is off by
// up to half an ulp, 0.004 rad at position 100,000 and 64 rad at 2^31; this is right
// to 2^-22 at every int32 position (frequencies up to 2^20). The rotation runs in
// 32 bits and is rounded once, to the cache's type.
//
// The work is moving 16-bit values once in and once out (HBM-bound; for a
// decode step of a few tokens it is launch latency). One CTA per token: its
// sines and cosines are shared by all heads.
#include "cascade_b200.h"
#include "internal.h"
#include "paged_device.cuh"

namespace cb {

int32_t* error_word();

struct AppendParams {
  const uint16_t *q, *k, *v;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;  // strides in elements
  const float* inv_freq;
  const int32_t *position, *sequence, *table;
  uint16_t *q_out, *k_pages, *v_pages;
  int q_heads, kv_heads, head_dim, rotary, interleaved;
  int sequences, table_width, pages, page_size;
  uint32_t item_mul;  // w / items = w * item_mul >> 32 for w < 2^22 (items <= 32); 0: items = 1
  float factor;
  int* err;
};

// Threads of a token's CTA: one wave of CTAs takes more (an item each at 48 heads
// of 128; 64 tokens 2.8 us, 3.8 with 128 threads), a long prompt fewer (8193
// tokens 35 us = 5.7 TB/s in a graph, 41 with 384).
constexpr int kAppendFew = 384, kAppendMany = 128;
constexpr int kMaxRotary = 512;
// 2 pi as a double and what it leaves out (2 pi = 6.283185307179586476925286766559005768...)
constexpr double kTurnHigh = 6.283185307179586, kTurnLow = 2.4492935982947064e-16, kTurnsPerRadian = 1.0 / kTurnHigh;

template <typename T>
__global__ void __launch_bounds__(kAppendFew) paged_append_kernel(const __grid_constant__ AppendParams p) {
  __shared__ float2 turn[kMaxRotary / 2];  // (cos, sin) of the token's angles
  grid_dep_wait();
  const int n = blockIdx.x;
  const int pos = p.position[n];
  // where the token goes: a negative position is padding (nothing is written
  // to the cache, q becomes zero)
  const int seq = p.sequence ? p.sequence[n] : n;
  int64_t row = -1;
  if (pos >= 0) {
    const int column = pos / p.page_size;
    int page = -1;
    if (seq >= 0 && seq < p.sequences && column < p.table_width)
      page = p.table[int64_t(seq) * p.table_width + column];
    if (page >= 0 && page < p.pages)
      row = int64_t(page) * p.kv_heads * p.page_size + pos % p.page_size;
    else if (threadIdx.x == 0 && p.err)
      atomicExch(p.err, kErrAppendIndex);
  }
  const int half = p.rotary >> 1;
  for (int i = threadIdx.x; i < half; i += blockDim.x) {
    const double f = double(p.inv_freq[i]), product = f * double(pos), rest = fma(f, double(pos), -product);
    const double turns = rint(product * kTurnsPerRadian);
    const double angle = fma(-turns, kTurnHigh, product) + fma(-turns, kTurnLow, rest);
    const float hi = float(angle), lo = float(angle - double(hi));
    float s, c;
    sincosf(hi, &s, &c);
    turn[i] = make_float2((c - s * lo) * p.factor, (s + c * lo) * p.factor);
  }
  __syncthreads();

  // an item is two 16-byte vectors of a head that are rotated together
  // (interleaved: 16 neighbours; half layout: 8 and their 8 partners)
  const int items = p.head_dim >> 4, rotated = p.rotary >> 4;
  const int heads = p.q_heads + 2 * p.kv_heads;
  for (int w = threadIdx.x; w < heads * items; w += blockDim.x) {
    int head = p.item_mul ? int(__umulhi(uint32_t(w), p.item_mul)) : w;
    const int j = w - head * items;
    const uint16_t* src;
    uint16_t* dst;
    bool turned = j < rotated, zero = false;
    if (head < p.q_heads) {
      src = p.q + n * p.q_token + head * p.q_head;
      dst = p.q_out + (int64_t(n) * p.q_heads + head) * p.head_dim;
      zero = pos < 0;
    } else {
      if (row < 0) continue;
      head -= p.q_heads;
      const bool value = head >= p.kv_heads;
      if (value) head -= p.kv_heads;
      turned = turned && !value;
      src = value ? p.v + n * p.v_token + head * p.v_head : p.k + n * p.k_token + head * p.k_head;
      dst = (value ? p.v_pages : p.k_pages) + (row + int64_t(head) * p.page_size) * p.head_dim;
    }
    const bool split = j < rotated && !p.interleaved;
    const int a = split ? j * 8 : j * 16;
    const int b = split ? half + j * 8 : j * 16 + 8;
    uint4 x = ld_cg_u4(src + a), y = ld_cg_u4(src + b);
    if (zero) {
      x = y = make_uint4(0, 0, 0, 0);
    } else if (turned) {
      uint32_t* xw = &x.x;
      uint32_t* yw = &y.x;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (split) {
          const float2 t0 = turn[a + 2 * e], t1 = turn[a + 2 * e + 1];
          const float x0 = T::lo(xw[e]), x1 = T::hi(xw[e]), y0 = T::lo(yw[e]), y1 = T::hi(yw[e]);
          xw[e] = T::pack(x0 * t0.x - y0 * t0.y, x1 * t1.x - y1 * t1.y);
          yw[e] = T::pack(y0 * t0.x + x0 * t0.y, y1 * t1.x + x1 * t1.y);
        } else {
          const float2 t0 = turn[j * 8 + e], t1 = turn[j * 8 + 4 + e];
          const float x0 = T::lo(xw[e]), x1 = T::hi(xw[e]), y0 = T::lo(yw[e]), y1 = T::hi(yw[e]);
          xw[e] = T::pack(x0 * t0.x - x1 * t0.y, x1 * t0.x + x0 * t0.y);
          yw[e] = T::pack(y0 * t1.x - y1 * t1.y, y1 * t1.x + y0 * t1.y);
        }
      }
    }
    *reinterpret_cast<uint4*>(dst + a) = x;
    *reinterpret_cast<uint4*>(dst + b) = y;
  }
}

}  // namespace cb

using namespace cb;

extern "C" int cb_paged_append(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token,
                               int64_t k_head, const void* v, int64_t v_token, int64_t v_head, int dtype, int tokens,
                               int q_heads, int kv_heads, int head_dim, const float* inv_freq, int rotary,
                               int interleaved, float factor, const int32_t* position, const int32_t* sequence,
                               const int32_t* table, int sequences, int table_width, void* q_out, void* k_pages,
                               void* v_pages, int pages, int page_size, void* stream) {
  const char* what = "cb_paged_append";
  CB_REQUIRE(dtype == CB_BF16 || dtype == CB_FP16, "%s: dtype must be bf16 or fp16", what);
  CB_REQUIRE(tokens >= 0, "%s: tokens=%d", what, tokens);
  CB_REQUIRE(q_heads >= 0 && kv_heads >= 1, "%s: q_heads=%d kv_heads=%d", what, q_heads, kv_heads);
  CB_REQUIRE(head_dim >= 16 && head_dim <= kMaxRotary && head_dim % 16 == 0,
             "%s: head_dim=%d must be a multiple of 16 up to %d", what, head_dim, kMaxRotary);
  CB_REQUIRE((int64_t(q_heads) + 2 * int64_t(kv_heads)) * (head_dim / 16) < (1 << 22), "%s: q_heads=%d kv_heads=%d",
             what, q_heads, kv_heads);
  CB_REQUIRE(rotary >= 0 && rotary <= head_dim && rotary % 16 == 0,
             "%s: rotary=%d must be a multiple of 16 up to head_dim", what, rotary);
  CB_REQUIRE(pages >= 1 && page_size >= 1 && sequences >= 1 && table_width >= 1,
             "%s: pages, page_size, sequences and table_width must be positive", what);
  if (tokens == 0) return kOk;
  CB_REQUIRE(k && v && position && table && k_pages && v_pages && (rotary == 0 || inv_freq) &&
                 (q_heads == 0 || (q && q_out)),
             "%s: null pointer", what);
  CB_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(q_out) && aligned16(k_pages) &&
                 aligned16(v_pages),
             "%s: q/k/v/q_out/pages must be 16-byte aligned", what);
  CB_REQUIRE((q_token | q_head | k_token | k_head | v_token | v_head) % 8 == 0,
             "%s: strides must be multiples of 8 elements", what);
  AppendParams p = {};
  p.q = static_cast<const uint16_t*>(q);
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.q_token = q_token, p.q_head = q_head;
  p.k_token = k_token, p.k_head = k_head;
  p.v_token = v_token, p.v_head = v_head;
  p.inv_freq = inv_freq;
  p.position = position, p.sequence = sequence, p.table = table;
  p.q_out = static_cast<uint16_t*>(q_out);
  p.k_pages = static_cast<uint16_t*>(k_pages);
  p.v_pages = static_cast<uint16_t*>(v_pages);
  const int items = head_dim / 16;
  p.item_mul = items == 1 ? 0 : uint32_t(((uint64_t(1) << 32) + items - 1) / items);
  p.q_heads = q_heads, p.kv_heads = kv_heads, p.head_dim = head_dim;
  p.rotary = rotary, p.interleaved = interleaved != 0, p.factor = factor;
  p.sequences = sequences, p.table_width = table_width, p.pages = pages, p.page_size = page_size;
  p.err = error_word();
  return launch(what, dtype == CB_BF16 ? paged_append_kernel<Bf16> : paged_append_kernel<Fp16>, dim3(tokens),
                dim3(tokens <= 4 * sm_count() ? kAppendFew : kAppendMany), 0, static_cast<cudaStream_t>(stream), p);
}
