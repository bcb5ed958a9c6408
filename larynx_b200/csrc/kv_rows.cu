// Writing rows into the 4-bit cache and reading them back.
//
// A warp takes one block (16 tokens) of one head, K and V.  Lane (n, j),
// n = lane / 4, j = lane % 4, works on tokens n and n + 8 and on channels
// 64 h + 32 w + 8 j + {0..7}: the codes that the lane holds of the K fragment,
// so K needs no exchange; V's codes pass through shared memory.  Both sides of
// memory move in pieces of 8 to 32 bytes a lane.
//
// Quantising, per token and group (include/larynx_kv.h): the codes are those
// of exact arithmetic.  x - m is taken with its rounding error (two-sum), the
// quotient from the reciprocal of s, and where the remainder d - c s comes
// within a hair of s / 2 the decision is made on the exact remainder.
#include <cfloat>

#include "kv.cuh"

namespace lx {
namespace kv {
namespace {

constexpr int WARPS = 4;
constexpr float MAGIC = 12582912.0f;  // 1.5 * 2^23: adding it rounds to an integer

__device__ __forceinline__ float min_nan(float a, float b) {
  float c;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
  return c;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float c;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
  return c;
}

// The rounding error of d = fl(a - b).
__device__ __forceinline__ float diff_error(float a, float b, float d) {
  const float bv = a - d, av = d + bv;
  return (a - av) - (b - bv);
}

// The bf16 value (as its 16 bits) at or below x.
__device__ __forceinline__ uint32_t bf16_floor(float x) {
  uint32_t u = __float_as_uint(x);
  if (u >> 31) u += 0xFFFFu;
  return u >> 16;
}

__device__ __forceinline__ float bf16_value(uint32_t u) { return __uint_as_float(u << 16); }

struct Params {
  float s, m, inv;
  uint32_t packed;  // bf16 s in the low half, bf16 m in the high half
};

// Step and minimum of a group with smallest and largest value lo, hi (NaN where
// the group holds one).  s is the least bf16 value with 15 s >= hi - m: the
// rounded quotient is at most one bf16 step off, and 15 s is exact in fp32.
__device__ __forceinline__ Params params_of(float lo, float hi) {
  Params p;
  const uint32_t mb = bf16_floor(lo);
  const float m = bf16_value(mb), range = hi - m;
  const float rest = diff_error(hi, m, range);
  if (!(fabsf(lo) <= FLT_MAX) || !(fabsf(m) <= FLT_MAX) || !(fabsf(hi) <= FLT_MAX) || !(range <= FLT_MAX)) {
    p.s = p.m = __uint_as_float(0x7fc00000u);
    p.inv = 0.0f;
    p.packed = 0x7fc07fc0u;
    return p;
  }
  constexpr uint32_t least = 0x00800000u;  // 2^-126
  uint32_t sb = (__float_as_uint(__fdiv_rn(range, 15.0f)) + 0xFFFFu) & 0xFFFF0000u;
  sb = sb < least ? least : sb;
  float top = 15.0f * __uint_as_float(sb);
  if (top < range || (top == range && rest > 0.0f)) {
    sb += 0x10000u;
  } else if (sb > least) {
    top = 15.0f * __uint_as_float(sb - 0x10000u);
    if (top > range || (top == range && rest <= 0.0f)) sb -= 0x10000u;
  }
  p.s = __uint_as_float(sb);
  p.m = m;
  p.inv = __frcp_rn(p.s);
  p.packed = (sb >> 16) | (mb << 16);
  return p;
}

// The code of x: rint((x - m) / s) in exact arithmetic, ties to even.  With
// c = rint(fl(x - m) / s), the remainder e = fl(x - m) - c s is exact (a multiple of the
// smaller ulp, at most about s / 2); only where |e| reaches s / 2 can the
// rounding of the quotient, or of x - m, have decided wrongly.
__device__ __forceinline__ uint32_t code_of(float x, const Params& p) {
  const float d = x - p.m;
  float t = fmaf(d, p.inv, MAGIC);
  float c = t - MAGIC;
  const float e = fmaf(-c, p.s, d);
  if (2.0f * fabsf(e) >= 0.99999f * p.s) {
    const float rest = diff_error(x, p.m, d), h = 0.5f * p.s;
    const bool odd = __float_as_uint(t) & 1u;
    if (e > h || (e == h && (rest > 0.0f || (rest == 0.0f && odd)))) c += 1.0f;
    if (e < -h || (e == -h && (rest < 0.0f || (rest == 0.0f && odd)))) c -= 1.0f;
    c = fminf(fmaxf(c, 0.0f), 15.0f);
    t = c + MAGIC;
  }
  return __float_as_uint(t) & 15u;
}

template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32(bf16 x) {
  return __bfloat162float(x);
}
template <>
__device__ __forceinline__ float to_f32(__half x) {
  return __half2float(x);
}
template <>
__device__ __forceinline__ float to_f32(float x) {
  return x;
}
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ bf16 from_f32(float x) {
  return __float2bfloat16_rn(x);
}
template <>
__device__ __forceinline__ __half from_f32(float x) {
  return __float2half_rn(x);
}
template <>
__device__ __forceinline__ float from_f32(float x) {
  return x;
}

// Eight neighbouring elements; `wide`: 16-byte aligned.
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool wide, float (&x)[8]) {
  if (wide) {
    constexpr int N = sizeof(T) / 2;
    uint4 u[N];
#pragma unroll
    for (int i = 0; i < N; ++i) u[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    const T* e = reinterpret_cast<const T*>(u);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(p[i]);
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, bool wide, const float (&x)[8]) {
  if (wide) {
    constexpr int N = sizeof(T) / 2;
    __align__(16) T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(x[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(e)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = from_f32<T>(x[i]);
  }
}

// What a warp works on: 16 tokens of one head of one entry.
struct Span {
  Entry e;
  int start, len, pos0, page;  // first position of the entry and of the block, the block's page
  size_t at;                   // its first byte
};

// The b-th block that entry i touches; false when there is none.
__device__ __forceinline__ bool span_of(const lx_kv_cache& c, const lx_kv_rows& r, int layer, int i, int b, int head,
                                        bool writes, Span& s) {
  s.e = entry_of(c, r, i);
  if (s.e.slot < 0 || s.e.rows == 0) return false;
  s.len = length_of(c, s.e.slot);
  s.start = start_of(r, i, s.len, s.e.rows);
  if (s.start == LX_KV_REFUSED) return false;  // an entry that was not served
  s.pos0 = (s.start & ~(BLOCK - 1)) + b * BLOCK;
  if (s.pos0 >= s.start + s.e.rows) return false;
  s.page = -1;
  if (s.pos0 >= 0 && s.pos0 < s.len) {
    s.page = c.table[static_cast<size_t>(s.e.slot) * c.max_pages + s.pos0 / c.page];
    if (s.page < 0 || s.page >= c.n_pages) {
      flag(c, LX_KV_PAGE);
      s.page = -1;
    } else {
      s.at = block_at(c, layer, s.page, head, s.pos0 % c.page / BLOCK);
      if (writes && c.refs[s.page] > 1) {  // held by a fork as well: lx_kv_extend gives a copy first
        flag(c, LX_KV_ROWS);
        s.page = -1;
      }
    }
  }
  return true;
}

template <typename T, int DIM, int GROUP>
__global__ void __launch_bounds__(32 * WARPS)
    k_kv_write(const lx_kv_cache c, int layer, const lx_kv_rows r, int blocks, const T* __restrict__ k, int64_t k_row,
               int64_t k_head, const T* __restrict__ v, int64_t v_row, int64_t v_head, bool wide) {
  constexpr int H = DIM / 64, G = DIM / GROUP;
  __shared__ __align__(16) uint16_t sv[WARPS][H * 256];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, n = lane / 4, j = lane % 4, head = blockIdx.y;
  const long long item = static_cast<long long>(blockIdx.x) * WARPS + warp;
  if (item >= static_cast<long long>(r.n) * blocks) return;
  Span s;
  if (!span_of(c, r, layer, static_cast<int>(item / blocks), static_cast<int>(item % blocks), head, true, s)) return;
  // tokens of the block that this entry writes (and that lie in the sequence)
  const int first = max(s.start - s.pos0, 0), past = min(min(s.start + s.e.rows, s.len) - s.pos0, BLOCK);
  if ((s.start < 0 || s.start + s.e.rows > s.len) && lane == 0) flag(c, LX_KV_ROWS);
  if (s.page < 0 || past <= first) return;
  uint8_t* block = static_cast<uint8_t*>(c.pool) + s.at;
  const bool full = first == 0 && past == BLOCK;
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    const T* src = kv ? v : k;
    const int64_t row_stride = kv ? v_row : k_row, head_stride = kv ? v_head : k_head;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      uint32_t word[2][2];  // [token n, n + 8][w]
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int t = n + 8 * u;
        const bool mine = t >= first && t < past;
        float x[2][8];
        const T* p = src + (s.e.row0 + (s.pos0 + t - s.start)) * row_stride + head * head_stride + 64 * h + 8 * j;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          if (mine)
            load8(p + 32 * w, wide, x[w]);
          else
#pragma unroll
            for (int i = 0; i < 8; ++i) x[w][i] = 0.0f;
        }
        float lo[2], hi[2];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          lo[w] = hi[w] = x[w][0];
#pragma unroll
          for (int i = 1; i < 8; ++i) {
            lo[w] = min_nan(lo[w], x[w][i]);
            hi[w] = max_nan(hi[w], x[w][i]);
          }
        }
        if (GROUP == 64) {
          lo[0] = lo[1] = min_nan(lo[0], lo[1]);
          hi[0] = hi[1] = max_nan(hi[0], hi[1]);
        }
#pragma unroll
        for (int w = 0; w < 64 / GROUP; ++w) {
#pragma unroll
          for (int o = 1; o < 4; o *= 2) {
            lo[w] = min_nan(lo[w], __shfl_xor_sync(0xffffffffu, lo[w], o));
            hi[w] = max_nan(hi[w], __shfl_xor_sync(0xffffffffu, hi[w], o));
          }
          const Params q = params_of(lo[w], hi[w]);
          const int g = 64 * h / GROUP + w;
          if (mine && j == 0)
            *reinterpret_cast<uint32_t*>(block + param_offset(DIM) + 64 * (kv * G + g) + 4 * param_slot(t)) = q.packed;
#pragma unroll
          for (int w2 = w; w2 < (GROUP == 64 ? 2 : w + 1); ++w2) {
            uint32_t bits = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const uint32_t code = code_of(x[w2][i], q);
              bits |= code << (kv ? 4 * i : 4 * (i / 2) + 16 * (i % 2));
            }
            word[u][w2] = bits;
          }
        }
      }
      if (!kv) {
        uint8_t* dst = block + 512 * h + 16 * lane;
        if (full) {
          *reinterpret_cast<uint4*>(dst) = make_uint4(word[0][0], word[0][1], word[1][0], word[1][1]);
        } else {
#pragma unroll
          for (int u = 0; u < 2; ++u)
            if (n + 8 * u >= first && n + 8 * u < past)
              *reinterpret_cast<uint2*>(dst + 8 * u) = make_uint2(word[u][0], word[u][1]);
        }
      } else {
        // V: lane (n', j') of the fragment takes tokens 2 j' + {0, 1, 8, 9}, channels 32 w + 4 n' + {0..3}
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int q = 0; q < 2; ++q)
              sv[warp][256 * h + ((2 * j + q) * 4 + n / 2) * 8 + 4 * u + 2 * w + n % 2] =
                  static_cast<uint16_t>(word[u][w] >> (16 * q));
      }
    }
  }
  __syncwarp();
#pragma unroll
  for (int h = 0; h < H; ++h) {
    uint8_t* dst = block + 512 * (H + h) + 16 * lane;
    const uint16_t* from = &sv[warp][256 * h + 8 * lane];
    if (full) {
      *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(from);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int t = 8 * (i / 4) + 2 * (lane % 4) + i % 2;
        if (t >= first && t < past) reinterpret_cast<uint16_t*>(dst)[i] = from[i];
      }
    }
  }
}

template <typename T, int DIM, int GROUP>
__global__ void __launch_bounds__(32 * WARPS)
    k_kv_read(const lx_kv_cache c, int layer, const lx_kv_rows r, int blocks, T* __restrict__ k, int64_t k_row,
              int64_t k_head, T* __restrict__ v, int64_t v_row, int64_t v_head, bool wide) {
  constexpr int H = DIM / 64, G = DIM / GROUP;
  __shared__ __align__(16) uint16_t sv[WARPS][H * 256];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, n = lane / 4, j = lane % 4, head = blockIdx.y;
  const long long item = static_cast<long long>(blockIdx.x) * WARPS + warp;
  if (item >= static_cast<long long>(r.n) * blocks) return;
  Span s;
  const int entry = static_cast<int>(item / blocks), b = static_cast<int>(item % blocks);
  if (!span_of(c, r, layer, entry, b, head, false, s)) {
    // a slot or an entry that does not exist: its rows read as 0
    if (s.e.rows == 0 || b * BLOCK >= s.e.rows || (s.e.slot >= 0 && s.start != LX_KV_REFUSED)) return;
    s.start = 0;
    s.pos0 = b * BLOCK;
    s.len = 0;
    s.page = -1;
  }
  const int first = max(s.start - s.pos0, 0), past = min(s.start + s.e.rows - s.pos0, BLOCK);
  const int held = s.page < 0 ? 0 : min(s.len - s.pos0, BLOCK);
  const uint8_t* block = static_cast<const uint8_t*>(c.pool) + (s.page < 0 ? 0 : s.at);
  uint4 kw[H];
#pragma unroll
  for (int h = 0; h < H; ++h) {
    kw[h] = make_uint4(0, 0, 0, 0);
    if (held > 0) {
      kw[h] = *reinterpret_cast<const uint4*>(block + 512 * h + 16 * lane);
      *reinterpret_cast<uint4*>(&sv[warp][256 * h + 8 * lane]) =
          *reinterpret_cast<const uint4*>(block + 512 * (H + h) + 16 * lane);
    }
  }
  __syncwarp();
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int t = n + 8 * u;
    if (t < first || t >= past) continue;
    const int64_t row = s.e.row0 + (s.pos0 + t - s.start);
#pragma unroll
    for (int kv = 0; kv < 2; ++kv)
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
          if (t < held) {
            const int g = (64 * h + 32 * w) / GROUP;
            const uint32_t p = *reinterpret_cast<const uint32_t*>(block + param_offset(DIM) + 64 * (kv * G + g) +
                                                                  4 * param_slot(t));
            const float step = bf16_value(p & 0xFFFFu), low = __uint_as_float(p & 0xFFFF0000u);
            uint32_t word;
            if (kv) {
              const uint16_t* from = &sv[warp][256 * h + (2 * j * 4 + n / 2) * 8 + 4 * u + 2 * w + n % 2];
              word = from[0] | static_cast<uint32_t>(from[32]) << 16;
            } else {
              word = u ? (w ? kw[h].w : kw[h].z) : (w ? kw[h].y : kw[h].x);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const uint32_t code = word >> (kv ? 4 * i : 4 * (i / 2) + 16 * (i % 2)) & 15u;
              x[i] = fmaf(static_cast<float>(code), step, low);
            }
          }
          T* dst = kv ? v + row * v_row + head * v_head : k + row * k_row + head * k_head;
          store8(dst + 64 * h + 32 * w + 8 * j, wide, x);
        }
  }
}

template <typename T>
bool wide_rows(const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head) {
  const int64_t per = 16 / static_cast<int64_t>(sizeof(T));
  return aligned(k, 16) && aligned(v, 16) && k_row % per == 0 && k_head % per == 0 && v_row % per == 0 &&
         v_head % per == 0;
}

template <typename T, int DIM, int GROUP>
bool go(bool writes, const lx_kv_cache& c, int layer, const lx_kv_rows& r, void* k, int64_t k_row, int64_t k_head,
        void* v, int64_t v_row, int64_t v_head, cudaStream_t s) {
  const int blocks = (r.max_rows + BLOCK - 1) / BLOCK + 1;  // rows may begin inside a block
  const long long items = static_cast<long long>(r.n) * blocks;
  const dim3 grid(static_cast<unsigned>((items + WARPS - 1) / WARPS), c.kv_heads);
  const bool wide = wide_rows<T>(k, k_row, k_head, v, v_row, v_head);
  if (writes)
    return launch(k_kv_write<T, DIM, GROUP>, grid, dim3(32 * WARPS), 0, s, c, layer, r, blocks,
                  static_cast<const T*>(k), k_row, k_head, static_cast<const T*>(v), v_row, v_head, wide);
  return launch(k_kv_read<T, DIM, GROUP>, grid, dim3(32 * WARPS), 0, s, c, layer, r, blocks, static_cast<T*>(k), k_row,
                k_head, static_cast<T*>(v), v_row, v_head, wide);
}

int rows_call(bool writes, const lx_kv_cache* c, int layer, const lx_kv_rows* r, int dtype, void* k, int64_t k_row,
              int64_t k_head, void* v, int64_t v_row, int64_t v_head, void* stream) {
  if (!cache_ok(c) || !rows_ok(r) || layer < 0 || layer >= c->n_layers || !k || !v) return LX_ERR_ARG;
  if (dtype != LX_KV_BF16 && dtype != LX_KV_FP16 && dtype != LX_KV_FP32) return LX_ERR_ARG;
  const size_t size = dtype == LX_KV_FP32 ? 4 : 2;
  if (!aligned(k, size) || !aligned(v, size)) return LX_ERR_ARG;
  const long long blocks = (static_cast<long long>(r->max_rows) + BLOCK - 1) / BLOCK + 1;
  if (blocks * r->n > (static_cast<long long>(0x7fffffff) - WARPS)) return LX_ERR_ARG;
  if (r->max_rows == 0 || r->total == 0) return LX_OK;
  OnDevice on(c->device);
  if (!on.ok()) return LX_ERR_CUDA;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int kind = dtype * 4 + (c->head_dim == 128) * 2 + (c->group == 64);
  bool ok = false;
#define LX_KV_CASE(N, T, D, G) \
  case N: ok = go<T, D, G>(writes, *c, layer, *r, k, k_row, k_head, v, v_row, v_head, s); break;
  switch (kind) {
    LX_KV_CASE(0, bf16, 64, 32)
    LX_KV_CASE(1, bf16, 64, 64)
    LX_KV_CASE(2, bf16, 128, 32)
    LX_KV_CASE(3, bf16, 128, 64)
    LX_KV_CASE(4, __half, 64, 32)
    LX_KV_CASE(5, __half, 64, 64)
    LX_KV_CASE(6, __half, 128, 32)
    LX_KV_CASE(7, __half, 128, 64)
    LX_KV_CASE(8, float, 64, 32)
    LX_KV_CASE(9, float, 64, 64)
    LX_KV_CASE(10, float, 128, 32)
    LX_KV_CASE(11, float, 128, 64)
  }
#undef LX_KV_CASE
  return ok ? LX_OK : LX_ERR_CUDA;
}

}  // namespace
}  // namespace kv
}  // namespace lx

extern "C" {

int lx_kv_write(const lx_kv_cache* c, int32_t layer, const lx_kv_rows* rows, int32_t dtype, const void* k,
                int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head, void* stream) {
  return lx::kv::rows_call(true, c, layer, rows, dtype, const_cast<void*>(k), k_row, k_head, const_cast<void*>(v),
                           v_row, v_head, stream);
}

int lx_kv_read(const lx_kv_cache* c, int32_t layer, const lx_kv_rows* rows, int32_t dtype, void* k, int64_t k_row,
               int64_t k_head, void* v, int64_t v_row, int64_t v_head, void* stream) {
  return lx::kv::rows_call(false, c, layer, rows, dtype, k, k_row, k_head, v, v_row, v_head, stream);
}

}  // extern "C"
