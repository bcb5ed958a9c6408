// Attention over the paged 4-bit cache (include/larynx_kv.h).
//
// Simple form: one CTA per (row, query head); thread i takes keys i, i + 128,
// ... with its own running maximum, sum and fp32 accumulators, which the CTA
// joins at the end.
#include <cmath>

#include "kv.cuh"

namespace lx {
namespace kv {
namespace {

constexpr int THREADS = 128;

struct Mask {
  int chunk, left;
  // keys [lo, hi) that a row at position p sees
  __device__ __forceinline__ void range(int p, int len, int& lo, int& hi) const {
    lo = 0;
    hi = len;
    if (chunk > 0) {
      int at = p / chunk;
      if (p < 0 && at * chunk != p) --at;  // rounds down
      const long long begin = static_cast<long long>(at) * chunk;
      hi = static_cast<int>(min(static_cast<long long>(len), begin + chunk));
      if (left >= 0) lo = static_cast<int>(max(0ll, begin - left));
    }
  }
};

template <typename T, int DIM, int GROUP>
__global__ void __launch_bounds__(THREADS)
    k_kv_attention(const lx_kv_cache c, int layer, const lx_kv_rows r, int q_heads, const T* __restrict__ q,
                   int64_t q_row, int64_t q_head, T* __restrict__ out, int64_t o_row, int64_t o_head, float* lse,
                   float scale, Mask mask) {
  constexpr int H = DIM / 64, G = DIM / GROUP;
  __shared__ float sq[DIM];
  __shared__ float sacc[4][DIM];
  __shared__ float sm[4], sl[4];
  const int i = blockIdx.x / r.max_rows, t = blockIdx.x % r.max_rows, h = blockIdx.y;
  const Entry e = entry_of(c, r, i);
  if (t >= e.rows) return;
  const int64_t row = e.row0 + t;
  const int head = h / (q_heads / c.kv_heads);
  for (int d = threadIdx.x; d < DIM; d += THREADS) sq[d] = static_cast<float>(q[row * q_row + h * q_head + d]);
  __syncthreads();
  int lo = 0, hi = 0;
  if (e.slot >= 0) {
    const int len = length_of(c, e.slot);
    const int start = start_of(r, i, len, e.rows);
    if (start != LX_KV_REFUSED) mask.range(start + t, len, lo, hi);
  }
  float m = -INFINITY, l = 0.0f, acc[DIM];
#pragma unroll
  for (int d = 0; d < DIM; ++d) acc[d] = 0.0f;
  for (int key = lo + static_cast<int>(threadIdx.x); key < hi; key += THREADS) {
    const int page = c.table[static_cast<size_t>(e.slot) * c.max_pages + key / c.page];
    if (page < 0 || page >= c.n_pages) {
      flag(c, LX_KV_PAGE);
      continue;
    }
    const uint8_t* b = static_cast<const uint8_t*>(c.pool) + block_at(c, layer, page, head, key % c.page / BLOCK);
    const int u = key % BLOCK;
    float s = 0.0f;
    for (int w = 0; w < DIM / 32; ++w) {
      const uint32_t par = *reinterpret_cast<const uint32_t*>(b + param_offset(DIM) + 64 * (32 * w / GROUP) + 4 * param_slot(u));
      const float step = __uint_as_float(par << 16), low = __uint_as_float(par & 0xFFFF0000u);
      for (int j = 0; j < 4; ++j) {
        const uint32_t word = *reinterpret_cast<const uint32_t*>(b + 512 * (w / 2) + 16 * (4 * (u % 8) + j) + 8 * (u / 8) + 4 * (w % 2));
        for (int x = 0; x < 8; ++x)
          s += sq[32 * w + 8 * j + x] * (static_cast<float>(word >> (4 * (x / 2) + 16 * (x % 2)) & 15u) * step + low);
      }
    }
    s *= scale;
    const float top = fmaxf(m, s), keep = m == -INFINITY ? 0.0f : expf(m - top), p = s == -INFINITY ? 0.0f : expf(s - top);
    l = l * keep + p;
    m = top;
#pragma unroll
    for (int w = 0; w < DIM / 32; ++w) {
      const uint32_t par = *reinterpret_cast<const uint32_t*>(b + param_offset(DIM) + 64 * (G + 32 * w / GROUP) + 4 * param_slot(u));
      const float step = __uint_as_float(par << 16), low = __uint_as_float(par & 0xFFFF0000u);
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const uint32_t word = *reinterpret_cast<const uint16_t*>(b + 512 * (H + w / 2) + 16 * (4 * n + u % 8 / 2) + 8 * (u / 8) + 4 * (w % 2) + 2 * (u % 2));
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          float& a = acc[32 * w + 4 * n + x];
          a = a * keep + p * (static_cast<float>(word >> (4 * x) & 15u) * step + low);
        }
      }
    }
  }
  // join the threads
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  float top = m;
  for (int o = 16; o; o /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) sm[warp] = top;
  __syncthreads();
  top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  const float f = m == -INFINITY ? (l == 0.0f ? 0.0f : l) : expf(m - top);  // (l is NaN where a score was)
  l *= f;
  for (int o = 16; o; o /= 2) l += __shfl_xor_sync(0xffffffffu, l, o);
  if (lane == 0) sl[warp] = l;
#pragma unroll
  for (int d = 0; d < DIM; ++d) {
    float a = acc[d] * f;
    for (int o = 16; o; o /= 2) a += __shfl_xor_sync(0xffffffffu, a, o);
    if (lane == 0) sacc[warp][d] = a;
  }
  __syncthreads();
  l = sl[0] + sl[1] + sl[2] + sl[3];
  for (int d = threadIdx.x; d < DIM; d += THREADS) {
    const float a = sacc[0][d] + sacc[1][d] + sacc[2][d] + sacc[3][d];
    out[row * o_row + h * o_head + d] = static_cast<T>(l == 0.0f ? 0.0f : a / l);
  }
  if (lse && threadIdx.x == 0) lse[row * q_heads + h] = l == 0.0f ? -INFINITY : top + logf(l);
}

struct Call {
  const lx_kv_cache* c;
  const lx_kv_rows* r;
  int layer, q_heads;
  const void* q;
  int64_t q_row, q_head;
  void* out;
  int64_t o_row, o_head;
  float* lse;
  float scale;
  Mask mask;
  int max_len;
  cudaStream_t s;
};

template <typename T, int DIM, int GROUP>
bool go(const Call& a) {
  const dim3 grid(static_cast<unsigned>(a.r->n) * static_cast<unsigned>(a.r->max_rows), a.q_heads);
  return launch(k_kv_attention<T, DIM, GROUP>, grid, dim3(THREADS), 0, a.s, *a.c, a.layer, *a.r, a.q_heads,
                static_cast<const T*>(a.q), a.q_row, a.q_head, static_cast<T*>(a.out), a.o_row, a.o_head, a.lse,
                a.scale, a.mask);
}

}  // namespace
}  // namespace kv
}  // namespace lx

extern "C" int lx_kv_attention(const lx_kv_cache* c, int32_t layer, const lx_kv_rows* rows, int32_t q_heads,
                               int32_t dtype, const void* q, int64_t q_row, int64_t q_head, void* out, int64_t o_row,
                               int64_t o_head, float* lse, float scale, int32_t chunk, int32_t left, int32_t max_len,
                               void* stream) {
  using namespace lx::kv;
  if (!cache_ok(c) || !rows_ok(rows) || layer < 0 || layer >= c->n_layers || !q || !out) return LX_ERR_ARG;
  if (dtype != LX_KV_BF16 && dtype != LX_KV_FP16) return LX_ERR_ARG;
  if (!aligned(q, 2) || !aligned(out, 2) || !aligned(lse, 4)) return LX_ERR_ARG;
  if (q_heads <= 0 || q_heads % c->kv_heads != 0 || q_heads > 65535) return LX_ERR_ARG;
  if (!std::isfinite(scale) || chunk < 0 || (chunk == 0 && left >= 0) || max_len < 0) return LX_ERR_ARG;
  if (static_cast<long long>(rows->n) * rows->max_rows > 0x7fffffff) return LX_ERR_ARG;
  if (rows->max_rows == 0 || rows->total == 0) return LX_OK;
  OnDevice on(c->device);
  if (!on.ok()) return LX_ERR_CUDA;
  const Call a{c,   rows, layer,  q_heads, q,       q_row, q_head, out,
               o_row, o_head, lse, scale, Mask{chunk, left}, max_len, static_cast<cudaStream_t>(stream)};
  bool ok = false;
  switch ((dtype == LX_KV_FP16) * 4 + (c->head_dim == 128) * 2 + (c->group == 64)) {
    case 0: ok = go<lx::bf16, 64, 32>(a); break;
    case 1: ok = go<lx::bf16, 64, 64>(a); break;
    case 2: ok = go<lx::bf16, 128, 32>(a); break;
    case 3: ok = go<lx::bf16, 128, 64>(a); break;
    case 4: ok = go<__half, 64, 32>(a); break;
    case 5: ok = go<__half, 64, 64>(a); break;
    case 6: ok = go<__half, 128, 32>(a); break;
    case 7: ok = go<__half, 128, 64>(a); break;
  }
  return ok ? LX_OK : LX_ERR_CUDA;
}
