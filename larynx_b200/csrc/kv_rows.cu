// Writing rows into the 4-bit cache and reading them back.
//
// A warp takes one block (16 tokens) of one head, K or V.  In writing, lane
// (n, j), n = lane / 4, j = lane % 4, works on tokens n and n + 8 and on channels
// 64 h + 32 w + 8 j + {0..7}: the codes that the lane holds of the K fragment,
// so K needs no exchange; V's codes pass through shared memory.  In reading, V is
// taken as it lies: lane (n, j) holds tokens 2 j + {0, 1, 8, 9} and channels
// 64 h + 32 w + 4 n + {0..3}.  All of a lane's loads are in flight before the first is used.
//
// Quantising, per token and group (include/larynx_kv.h): the codes are those
// of exact arithmetic.  x - m is taken with its rounding error (two-sum), the
// quotient from the reciprocal of s, and where one of eight remainders d - c s comes
// within a hair of s / 2 the decisions are made again on the exact remainders.
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
__device__ __forceinline__ float min_nan(float a, float b, float c) {
  float d;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float c;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
  return c;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
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

// rint((x - m) / s) + MAGIC in exact arithmetic, ties to even, given d = fl(x - m) and t, the same from the rounded quotient.
__device__ __noinline__ float exact_code(float x, float d, float t, float m, float s) {
  float c = t - MAGIC;
  const float e = fmaf(-c, s, d), rest = diff_error(x, m, d), h = 0.5f * s;
  const bool odd = __float_as_uint(t) & 1u;
  if (e > h || (e == h && (rest > 0.0f || (rest == 0.0f && odd)))) c += 1.0f;
  if (e < -h || (e == -h && (rest < 0.0f || (rest == 0.0f && odd)))) c -= 1.0f;
  return fminf(fmaxf(c, 0.0f), 15.0f) + MAGIC;
}

// The codes of eight values, code i at bit K ? 4 (i / 2) + 16 (i % 2) : 4 i.  With c = rint(fl(x - m) / s), the
// remainder e = fl(x - m) - c s is exact (a multiple of the smaller ulp, at most about s / 2); only where |e| reaches
// s / 2 can the rounding of the quotient, or of x - m, have decided wrongly.  MAGIC + c has c in its low bits, so a sum
// of products with powers of 16 packs the codes; what MAGIC adds is taken off at the end.
template <bool K>
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], const Params& p) {
  float d[8], t[8], far = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    d[i] = x[i] - p.m;
    t[i] = fmaf(d[i], p.inv, MAGIC);
    far = fmaxf(far, fabsf(fmaf(MAGIC - t[i], p.s, d[i])));
  }
  if (2.0f * far >= 0.99999f * p.s) {
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = exact_code(x[i], d[i], t[i], p.m, p.s);
  }
  uint32_t bits = 0, magic = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t by = 1u << (K ? 4 * (i / 2) + 16 * (i % 2) : 4 * i);
    bits += __float_as_uint(t[i]) * by;
    magic += 0x4B400000u * by;
  }
  return bits - magic;
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

// N neighbouring elements, N sizeof(T) a multiple of 8 bytes; `wide`: the address is as aligned as the widest access.
template <typename T, int N>
struct Pack {
  static constexpr int BYTES = N * static_cast<int>(sizeof(T));
  __align__(16) T e[BYTES >= 16 ? N : 16 / sizeof(T)];
  __device__ __forceinline__ void load(const T* p, bool wide) {
    if (wide) {
      if (BYTES == 8) {
        *reinterpret_cast<uint2*>(e) = __ldg(reinterpret_cast<const uint2*>(p));
      } else {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i)
          reinterpret_cast<uint4*>(e)[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) e[i] = p[i];
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = from_f32<T>(0.0f);
  }
  __device__ __forceinline__ void store(T* p, bool wide) const {
    if (wide) {
      if (BYTES == 8) {
        *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(e);
      } else {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(e)[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) p[i] = e[i];
    }
  }
};

// Codes 0..3 of a 16-bit field (the low half of `word`) as floats: with the exponent of 2^(23 - 4 i) above it, code i
// stands at the units of the float's mantissa.
__device__ __forceinline__ void codes_f32(uint32_t word, float (&c)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t one = static_cast<uint32_t>(127 + 23 - 4 * i) << 23;
    c[i] = __uint_as_float((word & (15u << (4 * i))) | one) - __uint_as_float(one);
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
  // the entry's words in flight together
  const int slot = r.seqs ? r.seqs[i] : i;
  const bool ok = slot >= 0 && slot < c.n_seq;
  const int length = c.lengths[ok ? slot : 0], given = r.start ? r.start[i] : 0;
  const int from = r.row0 ? r.row0[i] : 0, to = r.row0 ? r.row0[i + 1] : 0;
  s.e = entry_of(c, r, slot, from, to, i);
  s.start = 0;
  if (!ok || s.e.rows == 0) return false;
  s.len = clamp_length(c, length);
  s.start = clamp_start(r.start ? given : s.len - s.e.rows);
  if (s.start == LX_KV_REFUSED) return false;  // an entry that was not served
  s.pos0 = (s.start & ~(BLOCK - 1)) + b * BLOCK;
  if (s.pos0 >= s.start + s.e.rows) return false;
  s.page = -1;
  if (s.pos0 >= 0 && s.pos0 < s.len) {
    s.page = c.table[static_cast<size_t>(slot) * c.max_pages + s.pos0 / c.page];
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

// The block, head and side (K or V) of this warp.
struct Work {
  int entry, b, head, kv;
  bool any;
};
__device__ __forceinline__ Work work_of(const lx_kv_rows& r, int blocks) {
  Work w;
  const unsigned item = blockIdx.x * (WARPS / 2) + threadIdx.x / 64;
  w.entry = item / blocks;
  w.b = item - w.entry * blocks;
  w.head = blockIdx.y;
  w.kv = threadIdx.x / 32 % 2;
  w.any = w.entry < r.n;
  return w;
}

template <typename T, int DIM, int GROUP>
__global__ void __launch_bounds__(32 * WARPS)
    k_kv_write(const lx_kv_cache c, int layer, const lx_kv_rows r, int blocks, const T* __restrict__ k, int64_t k_row,
               int64_t k_head, const T* __restrict__ v, int64_t v_row, int64_t v_head, bool wide) {
  constexpr int H = DIM / 64, G = DIM / GROUP;
  __shared__ __align__(16) uint16_t sv[WARPS / 2][H * 256];
  const int pair = threadIdx.x / 64, lane = threadIdx.x % 32, n = lane / 4, j = lane % 4;
  pdl_launch_dependents();
  pdl_wait();
  const Work w = work_of(r, blocks);
  Span s;
  if (!w.any || !span_of(c, r, layer, w.entry, w.b, w.head, true, s)) return;
  // tokens of the block that this entry writes (and that lie in the sequence)
  const int first = max(s.start - s.pos0, 0), past = min(min(s.start + s.e.rows, s.len) - s.pos0, BLOCK);
  if ((s.start < 0 || s.start + s.e.rows > s.len) && lane == 0) flag(c, LX_KV_ROWS);
  if (s.page < 0 || past <= first) return;
  uint8_t* block = static_cast<uint8_t*>(c.pool) + s.at;
  const bool full = first == 0 && past == BLOCK;
  const T* src = w.kv ? v + w.head * v_head : k + w.head * k_head;
  const int64_t row = w.kv ? v_row : k_row;
  Pack<T, 8> raw[2][2 * H];  // tokens n, n + 8
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int t = n + 8 * u;
    const T* p = src + (s.e.row0 + (s.pos0 + t - s.start)) * row + 8 * j;
#pragma unroll
    for (int hw = 0; hw < 2 * H; ++hw) {
      if (t >= first && t < past)
        raw[u][hw].load(p + 32 * hw, wide);
      else
        raw[u][hw].clear();
    }
  }
  uint32_t word[2][2 * H];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int t = n + 8 * u;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      constexpr int PARTS = GROUP / 32;
      float x[PARTS][8], lo = 0.0f, hi = 0.0f;
#pragma unroll
      for (int q = 0; q < PARTS; ++q) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[q][i] = to_f32(raw[u][PARTS * g + q].e[i]);
        if (q == 0) lo = hi = x[0][0];
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          lo = min_nan(lo, x[q][i], x[q][i + 1]);
          hi = max_nan(hi, x[q][i], x[q][i + 1]);
        }
      }
#pragma unroll
      for (int o = 1; o < 4; o *= 2) {
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      }
      const Params p = params_of(lo, hi);
      if (j == 0 && t >= first && t < past)
        *reinterpret_cast<uint32_t*>(block + param_offset(DIM) + 64 * (w.kv * G + g) + 4 * param_slot(t)) = p.packed;
#pragma unroll
      for (int q = 0; q < PARTS; ++q)
        word[u][PARTS * g + q] = w.kv ? codes_of<false>(x[q], p) : codes_of<true>(x[q], p);
    }
  }
  if (!w.kv) {
#pragma unroll
    for (int h = 0; h < H; ++h) {
      uint8_t* dst = block + 512 * h + 16 * lane;
      if (full) {
        *reinterpret_cast<uint4*>(dst) =
            make_uint4(word[0][2 * h], word[0][2 * h + 1], word[1][2 * h], word[1][2 * h + 1]);
      } else {
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (n + 8 * u >= first && n + 8 * u < past)
            *reinterpret_cast<uint2*>(dst + 8 * u) = make_uint2(word[u][2 * h], word[u][2 * h + 1]);
      }
    }
    return;
  }
  // V: lane (n', j') of the fragment takes tokens 2 j' + {0, 1, 8, 9}, channels 32 w + 4 n' + {0..3}
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int hw = 0; hw < 2 * H; ++hw)
#pragma unroll
      for (int q = 0; q < 2; ++q)
        sv[pair][256 * (hw / 2) + ((2 * j + q) * 4 + n / 2) * 8 + 4 * u + 2 * (hw % 2) + n % 2] =
            static_cast<uint16_t>(word[u][hw] >> (16 * q));
  __syncwarp();
#pragma unroll
  for (int h = 0; h < H; ++h) {
    uint8_t* dst = block + 512 * (H + h) + 16 * lane;
    const uint16_t* from = &sv[pair][256 * h + 8 * lane];
    if (full) {
      *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(from);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int t = 8 * (i / 4) + 2 * j + i % 2;
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
  const int lane = threadIdx.x % 32, n = lane / 4, j = lane % 4;
  pdl_launch_dependents();
  pdl_wait();
  const Work w = work_of(r, blocks);
  if (!w.any) return;
  Span s;
  if (!span_of(c, r, layer, w.entry, w.b, w.head, false, s)) {
    // a slot or an entry that does not exist: its rows read as 0
    if (s.e.rows == 0 || w.b * BLOCK >= s.e.rows || (s.e.slot >= 0 && s.start != LX_KV_REFUSED)) return;
    s.start = 0;
    s.pos0 = w.b * BLOCK;
    s.len = 0;
    s.page = -1;
  }
  const int first = max(s.start - s.pos0, 0), past = min(s.start + s.e.rows - s.pos0, BLOCK);
  const int held = s.page < 0 ? 0 : min(s.len - s.pos0, BLOCK);
  const uint8_t* block = static_cast<const uint8_t*>(c.pool) + (s.page < 0 ? 0 : s.at);
  uint4 code[H];
#pragma unroll
  for (int h = 0; h < H; ++h)
    code[h] = held > 0 ? __ldcg(reinterpret_cast<const uint4*>(block + 512 * (w.kv * H + h) + 16 * lane))
                       : make_uint4(0, 0, 0, 0);
  T* dst = w.kv ? v + w.head * v_head : k + w.head * k_head;
  const int64_t row = w.kv ? v_row : k_row;
  const uint8_t* par = block + param_offset(DIM) + 64 * G * w.kv;
  if (!w.kv) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int t = n + 8 * u;
      if (t < first || t >= past) continue;
      T* out = dst + (s.e.row0 + (s.pos0 + t - s.start)) * row + 8 * j;
      uint32_t p[G];
#pragma unroll
      for (int g = 0; g < G; ++g)
        p[g] = t < held ? __ldcg(reinterpret_cast<const uint32_t*>(par + 64 * g + 4 * param_slot(t))) : 0u;
#pragma unroll
      for (int hw = 0; hw < 2 * H; ++hw) {
        const uint4 x = code[hw / 2];
        const uint32_t word = u ? (hw % 2 ? x.w : x.z) : (hw % 2 ? x.y : x.x);
        const float step = bf16_value(p[32 * hw / GROUP] & 0xFFFFu), low = __uint_as_float(p[32 * hw / GROUP] & 0xFFFF0000u);
        float even[4], odd[4];
        codes_f32(word, even);
        codes_f32(word >> 16, odd);
        Pack<T, 8> y;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y.e[2 * i] = from_f32<T>(fmaf(even[i], step, low));
          y.e[2 * i + 1] = from_f32<T>(fmaf(odd[i], step, low));
        }
        if (t >= held) y.clear();
        y.store(out + 32 * hw, wide);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = 2 * j + 8 * (i / 2) + i % 2;
    if (t < first || t >= past) continue;
    T* out = dst + (s.e.row0 + (s.pos0 + t - s.start)) * row + 4 * n;
    uint32_t p[G];
#pragma unroll
    for (int g = 0; g < G; ++g)
      p[g] = t < held ? __ldcg(reinterpret_cast<const uint32_t*>(par + 64 * g + 4 * param_slot(t))) : 0u;
#pragma unroll
    for (int hw = 0; hw < 2 * H; ++hw) {
      const uint4 x = code[hw / 2];
      const uint32_t word = i / 2 ? (hw % 2 ? x.w : x.z) : (hw % 2 ? x.y : x.x);
      const float step = bf16_value(p[32 * hw / GROUP] & 0xFFFFu), low = __uint_as_float(p[32 * hw / GROUP] & 0xFFFF0000u);
      float e[4];
      codes_f32(i % 2 ? word >> 16 : word, e);
      Pack<T, 4> y;
#pragma unroll
      for (int q = 0; q < 4; ++q) y.e[q] = from_f32<T>(t < held ? fmaf(e[q], step, low) : 0.0f);
      y.store(out + 32 * hw, wide);
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
  const int blocks = (r.max_rows + BLOCK - 2) / BLOCK + 1;  // rows may begin inside a block
  const long long items = static_cast<long long>(r.n) * blocks;
  const dim3 grid(static_cast<unsigned>((items + WARPS / 2 - 1) / (WARPS / 2)), c.kv_heads);
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
  const long long blocks = (static_cast<long long>(r->max_rows) + BLOCK - 2) / BLOCK + 1;
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
