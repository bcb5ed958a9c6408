// Attention over the paged 4-bit cache (include/larynx_kv.h) on the tensor cores.
//
// The codes go into the matrix instruction (m16n8k16, fp16 operands, fp32 sums)
// as they lie in memory: a 4-bit code c in the low mantissa bits of an fp16
// number is the subnormal c 2^-24 (16 c 2^-24 four bits further up), which the
// instruction multiplies exactly, so one AND makes two operands.  The steps and
// minima stay outside, in fp32: with k = c s + m per group of channels
//   q . k = s (q . c) + m sum(q)          (a scale per key, on the scores)
//   sum_j p_j v_j = sum_j (p_j s_j) (c_j - 8) + sum_j p_j (m_j + 8 s_j)  (a scale per key, on P)
// (The codes are centred for V because p s is rounded to fp16, which must not be
// multiplied by more than half the group's range: the product takes c, and a
// product with the constant 8 takes off what the centring needs, of the same
// rounded values.)
// q is scaled by a power of two so that its largest value is near 2^13 (an
// fp16 operand: what is lost is below 2^-38 of that); p s is scaled by a power
// of two F per group of channels that keeps it below 2^15 for the largest
// step seen so far and the largest p (2^4, see below), so that what fp16
// rounds away is 2^-11 of each term, or 2^-36 of the largest.
//
// A warp holds 16 rows (query rows x heads of one kv head) and walks the keys
// 32 at a time with a running maximum, sum and output in registers.  The maximum is raised, and the
// sums rescaled, only when a score exceeds it by 4 (log2 units): p <= 2^4.
// MW warps of a CTA hold different rows and share the keys' bytes, KW such
// groups split the CTA's keys, and a cluster of CTAs splits the keys of long
// sequences; they are joined through shared memory, in a fixed order.  The
// bytes come through rings of cp.async stages.
#include <cooperative_groups.h>

#include <cmath>

#include "kv.cuh"

namespace cg = cooperative_groups;

namespace lx {
namespace kv {
namespace {

constexpr int UNIT = 32;  // keys of a step: two blocks
constexpr uint32_t M0 = 0x000F000Fu, M1 = 0x00F000F0u;
constexpr float RAISE = 4.0f;        // log2 units by which a score may exceed the running maximum
constexpr float P_TOP = 2048.0f;     // F x the largest step: 2^4 x 2^11 stays below 2^15

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
      hi = static_cast<int>(max(0ll, min(static_cast<long long>(len), begin + chunk)));
      if (left >= 0) lo = static_cast<int>(max(0ll, begin - left));
    }
  }
};

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint4 lds128(const void* p) { return *reinterpret_cast<const uint4*>(p); }

// Steps and minima of two neighbouring keys from their parameter words.
__device__ __forceinline__ float2 steps(uint32_t a, uint32_t b) {
  return make_float2(__uint_as_float(a << 16), __uint_as_float(b << 16));
}
__device__ __forceinline__ float2 minima(uint32_t a, uint32_t b) {
  return make_float2(__uint_as_float(a & 0xFFFF0000u), __uint_as_float(b & 0xFFFF0000u));
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

template <int DIM, int GROUP, int MW, int KW>
struct Shape {
  static constexpr int THREADS = 32 * MW * KW;
  static constexpr int BB = block_bytes(DIM, GROUP);
  static constexpr int STAGES = DIM == 64 ? 4 : 3;
  static constexpr int RING = KW * STAGES * 2 * BB;
  static constexpr int ROWS = 16 * MW;
  // joining: per key group O [ROWS][DIM], m [ROWS], l [ROWS]; it takes the rings' place
  static constexpr int PART = ROWS * (DIM + 2) * 4;
  static constexpr int SMEM = (RING > (KW + 1) * PART ? RING : (KW + 1) * PART) + 16 * KW * STAGES;
};

template <typename T, int DIM, int GROUP, int MW, int KW>
__global__ void __launch_bounds__(32 * MW * KW)
    k_kv_attention(const lx_kv_cache c, int layer, const lx_kv_rows r, int q_heads, int per, int tiles, int split,
                   const T* __restrict__ q, int64_t q_row, int64_t q_head, bool wide, T* __restrict__ out,
                   int64_t o_row, int64_t o_head, float* lse, float scale, Mask mask) {
  using S = Shape<DIM, GROUP, MW, KW>;
  constexpr int H = DIM / 64, G = DIM / GROUP, BB = S::BB, STAGES = S::STAGES;
  extern __shared__ __align__(128) uint8_t smem[];
  int* held = reinterpret_cast<int*>(smem + S::SMEM - 16 * KW * STAGES);  // [KW][STAGES][4]: blocks of the stage that exist
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, n = lane / 4, j = lane % 4;
  const int mw = warp % MW, kg = warp / MW, gt = threadIdx.x % (32 * MW);
  const int rank = blockIdx.x % split;
  int item = blockIdx.x / split;
  const int head = item % c.kv_heads;
  item /= c.kv_heads;
  const int tile = item % tiles, entry = item / tiles;

  const Entry e = entry_of(c, r, entry);
  const int rows = e.rows * per, row0 = tile * S::ROWS;
  if (row0 >= rows) return;  // the whole cluster
  const int n_rows = min(S::ROWS, rows - row0);
  int len = 0, start = LX_KV_REFUSED;
  if (e.slot >= 0) {
    len = length_of(c, e.slot);
    start = start_of(r, entry, len, e.rows);
  }
  // keys of this lane's two rows, of the warp's rows (seen by one: [lo, hi), by all: [lo_all, hi_all)), of the CTA's
  int lo[2] = {0, 0}, hi[2] = {0, 0}, lo_all = 0, hi_all = 0, lo_cta = 0, hi_cta = 0;
  if (start != LX_KV_REFUSED) {
    int x;
#pragma unroll
    for (int u = 0; u < 2; ++u)
      mask.range(start + min(row0 + 16 * mw + n + 8 * u, rows - 1) / per, len, lo[u], hi[u]);
    mask.range(start + min(row0 + 16 * mw, rows - 1) / per, len, x, hi_all);
    mask.range(start + min(row0 + 16 * mw + 15, rows - 1) / per, len, lo_all, x);
    mask.range(start + row0 / per, len, lo_cta, x);
    mask.range(start + (row0 + n_rows - 1) / per, len, x, hi_cta);
  }

  // the query as A operands; lane (n, j): channels 64 h + 32 w + 8 j + {0..7} of rows n and n + 8
  uint32_t qa[H][2][2][4];
  float qs[2][G];
  float c1;
  {
    float x[2][H][2][8], top = 0.0f;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int row = min(row0 + 16 * mw + n + 8 * u, rows - 1);
      const T* p = q + (e.row0 + row / per) * q_row + (head * per + row % per) * q_head + 8 * j;
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          if (wide) {
            const uint4 v = *reinterpret_cast<const uint4*>(p + 64 * h + 32 * w);
            const T* t = reinterpret_cast<const T*>(&v);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[u][h][w][i] = static_cast<float>(t[i]);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[u][h][w][i] = static_cast<float>(p[64 * h + 32 * w + i]);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float a = fabsf(x[u][h][w][i]);
            top = a <= 3.4e38f ? fmaxf(top, a) : top;
          }
        }
    }
#pragma unroll
    for (int o = 1; o < 32; o *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    // 2^up x top lies in [2^13, 2^14)
    const int up = top > 0.0f ? min(max(13 - ilogbf(top), -110), 110) : 0;
    const float f = ldexpf(1.0f, up), f16 = f * 0.0625f, l2 = scale * 1.4426950408889634f;
    c1 = ldexpf(l2, 24 - up);
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int g = 0; g < G; ++g) qs[u][g] = 0.0f;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const float(&y)[8] = x[u][h][w];
          float sum = 0.0f;
#pragma unroll
          for (int i = 0; i < 8; ++i) sum += y[i];
          qs[u][(64 * h + 32 * w) / GROUP] += sum;
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            __half2 a = __floats2half2_rn(y[4 * s] * f, y[4 * s + 1] * f);
            qa[h][w][s][u] = *reinterpret_cast<uint32_t*>(&a);
            a = __floats2half2_rn(y[4 * s + 2] * f16, y[4 * s + 3] * f16);
            qa[h][w][s][2 + u] = *reinterpret_cast<uint32_t*>(&a);
          }
        }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int g = 0; g < G; ++g) {
        qs[u][g] += __shfl_xor_sync(0xffffffffu, qs[u][g], 1);
        qs[u][g] += __shfl_xor_sync(0xffffffffu, qs[u][g], 2);
        qs[u][g] *= l2;
      }
  }

  // the units of this key group: unit0, unit0 + KW, ... < unit1
  int unit0 = 0, unit1 = 0;
  if (hi_cta > lo_cta) {
    const int first = lo_cta / UNIT, count = (hi_cta + UNIT - 1) / UNIT - first;
    unit0 = first + static_cast<int>(static_cast<long long>(count) * rank / split);
    unit1 = first + static_cast<int>(static_cast<long long>(count) * (rank + 1) / split);
  }
  unit0 += kg;
  const int32_t* table = c.table + static_cast<size_t>(e.slot < 0 ? 0 : e.slot) * c.max_pages;
  const int per_page = c.page / BLOCK;  // blocks
  const uint8_t* pool = static_cast<const uint8_t*>(c.pool);
  uint8_t* ring = smem + kg * STAGES * 2 * BB;
  int* ring_held = held + kg * STAGES * 4;

  // page ids of the next unit to load, read one step ahead
  int next = unit0, page[2] = {-1, -1};
  auto look_up = [&] {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int block = 2 * next + b;
      page[b] = next < unit1 && block * BLOCK < hi_cta ? table[block / per_page] : -2;
    }
  };
  auto load = [&](int stage) {
    int got = 0;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      if (page[b] >= 0 && page[b] < c.n_pages) {
        got |= 1 << b;
        const uint8_t* src = pool + block_at(c, layer, page[b], head, (2 * next + b) % per_page);
        const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(ring + (2 * stage + b) * BB));
#pragma unroll
        for (int x = 0; x < (BB / 16 + 32 * MW - 1) / (32 * MW); ++x) {
          const int at = gt + 32 * MW * x;
          if (at < BB / 16) cp_async16(dst + 16 * at, src + 16 * at);
        }
      } else if (page[b] != -2 && gt == 0) {
        flag(c, LX_KV_PAGE);
      }
    }
    if (gt == 0) ring_held[4 * stage] = got;
    cp_async_commit();
    next += KW;
    look_up();
  };
  look_up();
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) load(i);

  float o[H][2][4][4], o8[G][4];  // o8: the rounded p s F times 8, the same in every column
#pragma unroll
  for (int g = 0; g < G; ++g) o8[g][0] = o8[g][1] = o8[g][2] = o8[g][3] = 0.0f;
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[h][w][i][x] = 0.0f;
  float m[2] = {-INFINITY, -INFINITY};    // running maxima
  float off[2] = {0.0f, 0.0f};            // what is subtracted from the scores: m, 0 while nothing was seen
  float2 l[2] = {both(0.0f), both(0.0f)}; // sums of p, over this lane's keys
  float2 z[2][G];                         // sums of p (m_v + 8 s_v)
  float vtop[G], vf[G];                   // power of two above the largest step of V so far, F
#pragma unroll
  for (int g = 0; g < G; ++g) {
    z[0][g] = z[1][g] = both(0.0f);
    vtop[g] = 0.0f;
    vf[g] = 1.0f;
  }

  int stage = 0;
  for (int unit = unit0; unit < unit1; unit += KW) {
    cp_async_wait<STAGES - 2>();
    if (MW == 1)
      __syncwarp();
    else
      asm volatile("bar.sync %0, %1;" ::"r"(1 + kg), "n"(32 * MW) : "memory");
    load((stage + STAGES - 1) % STAGES);
    const uint8_t* data = ring + 2 * stage * BB;
    const int got = ring_held[4 * stage];
    stage = stage + 1 == STAGES ? 0 : stage + 1;
    const int key0 = unit * UNIT;

    // scores, in log2 units: s[block][row][key half]
    float2 s[2][2][2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const uint8_t* d = data + b * BB;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float raw[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
        for (int hw = g * GROUP / 32; hw < (g + 1) * GROUP / 32; ++hw) {
          const uint2 k0 = *reinterpret_cast<const uint2*>(d + 512 * (hw / 2) + 16 * lane);
          const uint2 k1 = *reinterpret_cast<const uint2*>(d + 512 * (hw / 2) + 16 * lane + 8);
          const uint32_t w0 = hw % 2 ? k0.y : k0.x, w1 = hw % 2 ? k1.y : k1.x;
          mma(raw[0], qa[hw / 2][hw % 2][0], w0 & M0, w0 & M1);
          mma(raw[1], qa[hw / 2][hw % 2][0], w1 & M0, w1 & M1);
          mma(raw[0], qa[hw / 2][hw % 2][1], w0 >> 8 & M0, w0 >> 8 & M1);
          mma(raw[1], qa[hw / 2][hw % 2][1], w1 >> 8 & M0, w1 >> 8 & M1);
        }
        const uint4 kp = lds128(d + param_offset(DIM) + 64 * g + 16 * j);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const uint32_t p0 = t ? kp.z : kp.x, p1 = t ? kp.w : kp.y;
          const float2 ks = __fmul2_rn(steps(p0, p1), both(c1)), km = minima(p0, p1);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float2 base = g == 0 ? __fmul2_rn(both(qs[u][g]), km) : __ffma2_rn(both(qs[u][g]), km, s[b][u][t]);
            s[b][u][t] = __ffma2_rn(make_float2(raw[t][2 * u], raw[t][2 * u + 1]), ks, base);
          }
        }
      }
    }
    const bool part = got != 3 || key0 < lo_all || key0 + UNIT > hi_all;
    uint32_t seen = 0xFFFFu;  // bit 8 b + 4 u + 2 t + x
    if (part) {
      seen = 0;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int key = key0 + 16 * b + 8 * t + 2 * j + x;
              const bool in = (got >> b & 1) && key >= lo[u] && key < hi[u];
              seen |= static_cast<uint32_t>(in) << (8 * b + 4 * u + 2 * t + x);
              if (!in) (x ? s[b][u][t].y : s[b][u][t].x) = -INFINITY;
            }
    }
    // steps of V; a step that nobody sees does not count
    float2 vs[2][G][2], vm[2][G][2];
    bool raise = false;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const uint4 vp = lds128(data + b * BB + param_offset(DIM) + 64 * (G + g) + 16 * j);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const uint32_t p0 = t ? vp.z : vp.x, p1 = t ? vp.w : vp.y;
          vs[b][g][t] = steps(p0, p1);
          vm[b][g][t] = __ffma2_rn(vs[b][g][t], both(8.0f), minima(p0, p1));
          if (part) {
            const uint32_t any = seen >> (8 * b + 2 * t) | seen >> (8 * b + 2 * t + 4);
            if (!(any & 1)) vs[b][g][t].x = vm[b][g][t].x = 0.0f;
            if (!(any & 2)) vs[b][g][t].y = vm[b][g][t].y = 0.0f;
          }
          raise |= fmaxf(vs[b][g][t].x, vs[b][g][t].y) > vtop[g];
        }
      }
    float top[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      top[u] = fmaxf(fmaxf(fmaxf(s[0][u][0].x, s[0][u][0].y), fmaxf(s[0][u][1].x, s[0][u][1].y)),
                     fmaxf(fmaxf(s[1][u][0].x, s[1][u][0].y), fmaxf(s[1][u][1].x, s[1][u][1].y)));
      raise |= top[u] > m[u] + RAISE;
    }
    if (__any_sync(0xffffffffu, raise)) {
      float f[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        top[u] = fmaxf(top[u], __shfl_xor_sync(0xffffffffu, top[u], 1));
        top[u] = fmaxf(top[u], __shfl_xor_sync(0xffffffffu, top[u], 2));
        const float to = fmaxf(m[u], top[u]);
        f[u] = to == -INFINITY ? 1.0f : ex2(m[u] - to);
        m[u] = to;
        off[u] = to == -INFINITY ? 0.0f : to;
        l[u] = __fmul2_rn(l[u], both(f[u]));
#pragma unroll
        for (int g = 0; g < G; ++g) z[u][g] = __fmul2_rn(z[u][g], both(f[u]));
      }
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float v = 0.0f;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int t = 0; t < 2; ++t) v = fmaxf(v, fmaxf(vs[b][g][t].x, vs[b][g][t].y));
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
        float ratio = 1.0f;
        if (v > vtop[g]) {  // the power of two at or above v, at least 2^-110
          const uint32_t bits = (__float_as_uint(v) + 0x7FFFFFu) & 0x7F800000u;
          const float to = fminf(fmaxf(__uint_as_float(bits), 7.7037198e-34f), 8.5070592e37f);
          const float nf = P_TOP / to;
          ratio = vtop[g] == 0.0f ? 1.0f : nf / vf[g];
          vtop[g] = v > to ? INFINITY : to;
          vf[g] = nf;
        }
#pragma unroll
        for (int hw = g * GROUP / 32; hw < (g + 1) * GROUP / 32; ++hw)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[hw / 2][hw % 2][i][x] *= f[x / 2] * ratio;
#pragma unroll
        for (int x = 0; x < 4; ++x) o8[g][x] *= f[x / 2] * ratio;
      }
    }
    // p, its sums, and O += (p s F) c
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const uint8_t* d = data + b * BB + 512 * H;
      float2 p[2][2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const float2 y = __fadd2_rn(s[b][u][t], both(-off[u]));
          p[u][t] = make_float2(ex2(y.x), ex2(y.y));
          l[u] = __fadd2_rn(l[u], p[u][t]);
        }
#pragma unroll
      for (int g = 0; g < G; ++g) {
        uint32_t pa[4];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const float2 f = __fmul2_rn(vs[b][g][t], both(vf[g]));
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float2 a = __fmul2_rn(p[u][t], f), add = p[u][t];
            if (part) {  // a key that this row does not see: not even its NaN counts
              const uint32_t in = seen >> (8 * b + 4 * u + 2 * t);
              float2 low = vm[b][g][t];
              if (!(in & 1)) a.x = low.x = 0.0f;
              if (!(in & 2)) a.y = low.y = 0.0f;
              z[u][g] = __ffma2_rn(add, low, z[u][g]);
            } else {
              z[u][g] = __ffma2_rn(add, vm[b][g][t], z[u][g]);
            }
            const __half2 hp = __float22half2_rn(a);
            pa[2 * t + u] = *reinterpret_cast<const uint32_t*>(&hp);
          }
        }
        mma(o8[g], pa, 0x00080008u, 0x00080008u);
#pragma unroll
        for (int hw = g * GROUP / 32; hw < (g + 1) * GROUP / 32; ++hw) {
          const uint4 v = lds128(d + 512 * (hw / 2) + 16 * lane);
          const uint32_t w0 = hw % 2 ? v.y : v.x, w1 = hw % 2 ? v.w : v.z;
          float(&acc)[4][4] = o[hw / 2][hw % 2];
          mma(acc[0], pa, w0 & M0, w1 & M0);
          mma(acc[1], pa, w0 & M1, w1 & M1);
          mma(acc[2], pa, w0 >> 8 & M0, w1 >> 8 & M0);
          mma(acc[3], pa, w0 >> 8 & M1, w1 >> 8 & M1);
        }
      }
    }
  }
  cp_async_wait<0>();
  __syncthreads();  // every ring has been read: the joining takes their place

  // this warp's result: O in true units
  float* part_o = reinterpret_cast<float*>(smem);              // [KW + 1][ROWS][DIM], the last one the CTA's
  float* part_m = part_o + (KW + 1) * S::ROWS * DIM;           // [KW + 1][ROWS]
  float* part_l = part_m + (KW + 1) * S::ROWS;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int row = 16 * mw + n + 8 * u;
    float sum = l[u].x + l[u].y;
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    if (j == 0) {
      part_m[kg * S::ROWS + row] = m[u];
      part_l[kg * S::ROWS + row] = sum;
    }
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const int g = (64 * h + 32 * w) / GROUP;
        float low = z[u][g].x + z[u][g].y;
        low += __shfl_xor_sync(0xffffffffu, low, 1);
        low += __shfl_xor_sync(0xffffffffu, low, 2);
        const float f = 1.0f / vf[g];
        // columns 2 j, 2 j + 1 of product i are channels 8 j + i and 8 j + 4 + i
        float* dst = part_o + (kg * S::ROWS + row) * DIM + 64 * h + 32 * w + 8 * j;
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            dst[4 * x + i] =
                fmaf((o[h][w][i][2 * u + x] * (i % 2 ? 0.0625f : 1.0f) - o8[g][2 * u + x]) * 16777216.0f, f, low);
      }
  }
  __syncthreads();
  // join the CTA's key groups
  float* cta_o = part_o + KW * S::ROWS * DIM;
  float* cta_m = part_m + KW * S::ROWS;
  float* cta_l = part_l + KW * S::ROWS;
  for (int x = threadIdx.x; x < n_rows * DIM; x += S::THREADS) {
    const int row = x / DIM;
    float top = part_m[row];
#pragma unroll
    for (int k = 1; k < KW; ++k) top = fmaxf(top, part_m[k * S::ROWS + row]);
    float a = 0.0f, sum = 0.0f;
#pragma unroll
    for (int k = 0; k < KW; ++k) {
      const float mk = part_m[k * S::ROWS + row];
      const float f = mk == top ? 1.0f : ex2(mk - top);
      a = fmaf(part_o[k * S::ROWS * DIM + x], f, a);
      sum = fmaf(part_l[k * S::ROWS + row], f, sum);
    }
    cta_o[x] = a;
    if (x % DIM == 0) {
      cta_m[row] = top;
      cta_l[row] = sum;
    }
  }
  if (split > 1)
    cg::this_cluster().sync();
  else
    __syncthreads();
  // join the cluster's CTAs, each a part of the outputs
  for (int x = threadIdx.x + rank * S::THREADS; x < n_rows * DIM; x += split * S::THREADS) {
    const int row = x / DIM, d = x % DIM;
    float top, a, sum;
    if (split > 1) {
      top = -INFINITY;
      for (int k = 0; k < split; ++k) top = fmaxf(top, *cg::this_cluster().map_shared_rank(cta_m + row, k));
      a = sum = 0.0f;
      for (int k = 0; k < split; ++k) {
        const float mk = *cg::this_cluster().map_shared_rank(cta_m + row, k);
        const float f = mk == top ? 1.0f : ex2(mk - top);
        a = fmaf(*cg::this_cluster().map_shared_rank(cta_o + x, k), f, a);
        sum = fmaf(*cg::this_cluster().map_shared_rank(cta_l + row, k), f, sum);
      }
    } else {
      top = cta_m[row];
      a = cta_o[x];
      sum = cta_l[row];
    }
    const int t = (row0 + row) / per, h = head * per + (row0 + row) % per;
    out[(e.row0 + t) * o_row + h * o_head + d] = static_cast<T>(sum == 0.0f ? 0.0f : a / sum);
    if (lse && d == 0)
      lse[static_cast<int64_t>(e.row0 + t) * q_heads + h] =
          sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
  }
  if (split > 1) cg::this_cluster().sync();  // nobody leaves while its part may be read
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

template <typename T, int DIM, int GROUP, int MW, int KW>
bool run(const Call& a) {
  using S = Shape<DIM, GROUP, MW, KW>;
  auto kernel = k_kv_attention<T, DIM, GROUP, MW, KW>;
  static bool ready[64] = {false};
  int dev = a.c->device & 63;
  if (!ready[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM) != cudaSuccess ||
        cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
      return false;
    ready[dev] = true;
  }
  const int per = a.q_heads / a.c->kv_heads;
  const long long tiles = (static_cast<long long>(a.r->max_rows) * per + S::ROWS - 1) / S::ROWS;
  const long long items = tiles * a.r->n * a.c->kv_heads;
  // split the keys over a cluster until the GPU is full, leaving each key group two steps
  const int most = a.max_len > 0 ? a.max_len : a.c->max_pages * a.c->page;
  int split = 1;
  while (split < 16 && items * split < 2 * num_sms() && most / UNIT >= 2 * KW * 2 * split) split *= 2;
  if (items * split > 0x7fffffff) return false;
  const bool wide = aligned(a.q, 16) && a.q_row % 8 == 0 && a.q_head % 8 == 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(items * split));
  cfg.blockDim = dim3(S::THREADS);
  cfg.dynamicSmemBytes = S::SMEM;
  cfg.stream = a.s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = split > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, *a.c, a.layer, *a.r, a.q_heads, per, static_cast<int>(tiles), split,
                            static_cast<const T*>(a.q), a.q_row, a.q_head, wide, static_cast<T*>(a.out), a.o_row,
                            a.o_head, a.lse, a.scale, a.mask) == cudaSuccess;
}

template <typename T, int DIM, int GROUP>
bool go(const Call& a) {
  const long long rows = static_cast<long long>(a.r->max_rows) * (a.q_heads / a.c->kv_heads);
  if (rows <= 16) return run<T, DIM, GROUP, 1, 4>(a);
  if (rows <= 32) return run<T, DIM, GROUP, 2, 2>(a);
  return run<T, DIM, GROUP, 4, 1>(a);
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
