// Root-mean-square norm with the residual's addition (rows in 16 / 32 bits, or e4m3 rows with a
// scale for each 128 columns), its gradients, and the quantisation to e4m3 blocks.
//
//   h = x + residual,  r = 1 / sqrt(mean(h^2) + eps),  y = h r w
//   quantised: per block of 128 columns  top = max(|y|, 2^-117),  scale = top / 448,
//              q = e4m3(y * (448 / top))
//   backward:  g = dy w,  n = h r,  dx = r (g - n mean(g n)) (+ dh),  dw = sum over rows of dy n
//
// All of them are bound by memory (4-14 operations a value).  A row lives in the registers of
// the T lanes that own it between its one read and its one write; every statistic is f32.
// At 204800 x 512 bf16 with the residual the norm takes 142 us (5.9 TB/s, a large copy 5.3), in f32 162
// without it (5.2) and 339 with it (5.0); its 8-bit form 135 with it (5.4), 96 without (3.3: a row's loads, its sums
// and its stores follow one another, and what is in flight no longer covers them).  Gradients of 100352 x 512 with
// their forward: bf16 41 + 58 + 4 us (5.0 TB/s), f32 73 + 125 + 5 (5.1).  204800 x 1024 quantised 133 us (4.8); 128 x
// 128 blocks of 5003 x 1111 f32 12.6 us (2.2: each workgroup loads one block, joins and stores it), of 4096 x 4096
// bf16 11.5 (4.4).  256 x 512 to 8 bits takes 3.7 us, a launch more than that.
// The gradient is taken at the stored h (rounded to x's type) with the r of the unrounded sum.
#include <type_traits>

#include "trk_common.h"

using namespace trk;

namespace {

typedef float f8v __attribute__((ext_vector_type(8)));
typedef _Float16 h2v __attribute__((ext_vector_type(2)));

constexpr float kTop = 448.0f;             // largest e4m3 value
constexpr float kLeast = 0x1p-117f;        // 448 / kLeast and kLeast / 448 are both normal f32
constexpr int kV = 8;                      // values of a vector (16 B of bf16)

template <int DT> struct El;
template <> struct El<TRK_F32> { typedef float T; };
template <> struct El<TRK_BF16> { typedef uint16_t T; };
template <> struct El<TRK_F16> { typedef uint16_t T; };

template <int DT>
__device__ __forceinline__ float to_f(typename El<DT>::T v) {
  if constexpr (DT == TRK_F32) return v;
  else if constexpr (DT == TRK_BF16) return __uint_as_float((uint32_t)v << 16);
  else return (float)__builtin_bit_cast(_Float16, v);
}

template <int DT>
__device__ __forceinline__ typename El<DT>::T from_f(float v) {
  if constexpr (DT == TRK_F32) return v;
  else if constexpr (DT == TRK_BF16) return f32_to_bf16(v);
  else return __builtin_bit_cast(uint16_t, (_Float16)v);
}

// 8 values at p, of which `left` exist; `row` values of the row lie before and including them.  Whole
// vectors are one or two 16-byte accesses: gfx950 takes them at any byte alignment.  A row's last,
// partial vector is the row's last 8 values, shifted down (value by value it took most of the time
// of rows of 500: 214 us for 204800 rows with the residual, now 171; 117 for rows of 512).
template <int DT>
__device__ __forceinline__ void load8(const typename El<DT>::T* p, int64_t left, int64_t row, float (&v)[kV]) {
  typename El<DT>::T t[kV];
  if (left >= kV) {
    __builtin_memcpy(t, p, sizeof t);
#pragma unroll
    for (int j = 0; j < kV; ++j) v[j] = to_f<DT>(t[j]);
  } else if (left > 0 && row >= kV) {
    const int s = kV - (int)left;
    __builtin_memcpy(t, p - s, sizeof t);
#pragma unroll
    for (int j = 0; j < kV; ++j) v[j] = to_f<DT>(t[j]);
#pragma unroll
    for (int d = 4; d > 0; d >>= 1)
      if (s & d)
#pragma unroll
        for (int j = 0; j < kV; ++j) v[j] = j + d < kV ? v[j + d] : 0.0f;
  } else {
#pragma unroll
    for (int j = 0; j < kV; ++j) v[j] = j < left ? to_f<DT>(p[j]) : 0.0f;
  }
}

template <int DT>
__device__ __forceinline__ void store8(typename El<DT>::T* p, int64_t left, const float (&v)[kV]) {
  typename El<DT>::T t[kV];
  if constexpr (DT == TRK_F32) {
    __builtin_memcpy(t, v, sizeof t);
  } else {
    uint32_t u[kV / 2];
#pragma unroll
    for (int j = 0; j < kV / 2; ++j) {
      if constexpr (DT == TRK_BF16) u[j] = pack2_bf16(v[2 * j], v[2 * j + 1]);
      else u[j] = __builtin_bit_cast(uint32_t, h2v{(_Float16)v[2 * j], (_Float16)v[2 * j + 1]});
    }
    __builtin_memcpy(t, u, sizeof t);
  }
  if (left >= kV) {
    __builtin_memcpy(p, t, sizeof t);
  } else if (left > 0) {  // a run of 4, of 2 and of 1
    constexpr int E = sizeof(t[0]);
    if (left & 4) __builtin_memcpy(p, t, 4 * E);
    if (left & 2) {
      if (left & 4) __builtin_memcpy(p + 4, t + 4, 2 * E);
      else __builtin_memcpy(p, t, 2 * E);
    }
    if (left & 1) {
#pragma unroll
      for (int j = 0; j < kV; j += 2)
        if (left == j + 1) p[j] = t[j];
    }
  }
}

// 8 f32 -> 8 e4m3 (round to nearest even; |v| <= 448 (1 + 2^-22) rounds to 448 at most; NaN stays)
__device__ __forceinline__ uint2 pack8_e4m3(const float (&v)[kV]) {
  int a = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
  a = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], a, true);
  int b = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], 0, false);
  b = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], b, true);
  return make_uint2((uint32_t)a, (uint32_t)b);
}

// 8 codes at p, of which `left` are values of the row; the `room` bytes there include the row's
// padding, which is written as zeros
__device__ __forceinline__ void store8_e4m3(uint8_t* p, int64_t left, int64_t room, uint2 c) {
  uint64_t w = (uint64_t)c.y << 32 | c.x;
  if (left < kV) w &= left > 0 ? ~0ull >> (64 - 8 * left) : 0;
  if (room >= kV) {
    __builtin_memcpy(p, &w, 8);
  } else {
#pragma unroll
    for (int j = 0; j < kV; ++j)
      if (j < room) p[j] = (uint8_t)(w >> (8 * j));
  }
}

template <int W>
__device__ __forceinline__ float sum_lanes(float v) {
#pragma unroll
  for (int m = 1; m < W; m <<= 1) v += __shfl_xor(v, m, kWave);
  return v;
}
template <int W>
__device__ __forceinline__ float max_lanes(float v) {
#pragma unroll
  for (int m = 1; m < W; m <<= 1) v = fmaxf(v, __shfl_xor(v, m, kWave));
  return v;
}

// sum over the T threads that own a row (T <= 64: lanes of one wave; else the workgroup, and
// every thread of it calls).  red: one float per wave.
template <int T>
__device__ __forceinline__ float sum_row(float v, float* red) {
  v = sum_lanes<(T < kWave ? T : kWave)>(v);
  if constexpr (T > kWave) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < T / kWave; ++w) v += red[w];
  }
  return v;
}

struct NormArgs {
  const void *x, *res, *weight;
  void *y, *h;         // y: rows of the input's type, or e4m3 codes
  float *rstd, *scale;
  int64_t ldx, ldr, ldy, ldh, sld, R, D;
  float eps;
};

// 448 / top as a sum of two f32 (with one, 1.5 u off, 2 to 3 times as many f32 values fell to the other
// side of a tie), so that v * (448 / top) is rounded once (to within 2^-40): values that
// lie halfway between two codes, common among 16-bit inputs, stay there and go to the even one.  An
// infinite top gives 0 (and NaN for the infinity itself).
struct Ratio {
  float hi, lo;
  __device__ __forceinline__ explicit Ratio(float top) {
    hi = kTop / top;
    const float rest = fmaf(-hi, top, kTop);  // exact
    lo = top < INFINITY ? rest / top : 0.0f;
  }
  __device__ __forceinline__ float operator*(float v) const { return fmaf(v, hi, v * lo); }
};

// quantise the 8 values a lane holds of its 128-column block (16 consecutive lanes)
__device__ __forceinline__ void quant8(const float (&v)[kV], uint8_t* q, int64_t col, int64_t D, int64_t ldq,
                                       float* scale) {
  float top = 0.0f;
#pragma unroll
  for (int j = 0; j < kV; ++j) top = fmaxf(top, fabsf(v[j]));
  top = fmaxf(max_lanes<16>(top), kLeast);
  const Ratio inv(top);
  float t[kV];
#pragma unroll
  for (int j = 0; j < kV; ++j) t[j] = inv * v[j];
  const int64_t pad = (D + 15) / 16 * 16;
  const int64_t room = (ldq >= pad ? pad : D) - col;  // the row's padding (to 16 bytes) is written as zeros
  if (room > 0) store8_e4m3(q + col, D - col, room, pack8_e4m3(t));
  if ((threadIdx.x & 15) == 0 && col < D) *scale = top / kTop;
}

// T threads own a row and hold it as NV vectors of 8; BT threads a workgroup.  Rows longer than
// T * NV * 8 (LOOP) are read twice.
template <int DT, int T, int NV, int BT, bool FP8, bool LOOP>
__global__ __launch_bounds__(BT) void rms_norm_kernel(NormArgs A) {
  typedef typename El<DT>::T E;
  __shared__ float red[BT / kWave];
  const int t = threadIdx.x % T;
  const int64_t row = (int64_t)blockIdx.x * (BT / T) + threadIdx.x / T;
  const bool on = row < A.R;  // T > 64: uniform over the workgroup (one row each)
  const int64_t rr = on ? row : 0;
  const E* x = (const E*)A.x + rr * A.ldx;
  const E* res = A.res ? (const E*)A.res + rr * A.ldr : nullptr;
  const int64_t D = on ? A.D : 0;
  float v[NV][kV];
  float ss = 0.0f;
  auto fetch = [&](int64_t c, float (&u)[kV]) {
    load8<DT>(x + c, D - c, D, u);
    if (res) {
      float w[kV];
      load8<DT>(res + c, D - c, D, w);
#pragma unroll
      for (int j = 0; j < kV; ++j) u[j] += w[j];
    }
  };
  const int64_t step = (int64_t)T * NV * kV;
  for (int64_t base = 0; base < (LOOP ? A.D : 1); base += step) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t c = base + (int64_t)(i * T + t) * kV;
      fetch(c, v[i]);
#pragma unroll
      for (int j = 0; j < kV; ++j) ss = fmaf(v[i][j], v[i][j], ss);
    }
  }
  ss = sum_row<T>(ss, red);
  const float r = 1.0f / sqrtf(ss / (float)A.D + A.eps);
  if (on && t == 0 && A.rstd) A.rstd[row] = r;
  for (int64_t base = 0; base < (LOOP ? A.D : 1); base += step) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t c = base + (int64_t)(i * T + t) * kV;
      if constexpr (LOOP) fetch(c, v[i]);
      if (A.h && c < D) store8<DT>((E*)A.h + rr * A.ldh + c, D - c, v[i]);
      float w[kV];
      if (A.weight) load8<DT>((const E*)A.weight + c, D - c, D, w);
#pragma unroll
      for (int j = 0; j < kV; ++j) v[i][j] = A.weight ? v[i][j] * r * w[j] : v[i][j] * r;
      if constexpr (FP8)
        quant8(v[i], (uint8_t*)A.y + rr * A.ldy, c, D, A.ldy, A.scale + (c >> 7) * A.sld + rr);
      else if (c < D)
        store8<DT>((E*)A.y + rr * A.ldy + c, D - c, v[i]);
    }
  }
}

struct BwdArgs {
  const void *h, *weight, *dy, *dh;
  const float* rstd;
  void *dx, *dw;
  float* part;
  int64_t ldh, ldy, lddh, ldx, R, D, parts;
};

// dx (null: not wanted) of the rows of workgroup blockIdx.x, blockIdx.x + gridDim.x, ..; part[blockIdx.x][D]
// its sum of dy n over those rows.  (T, NV, LOOP as above.)
template <int DT, int T, int NV, int BT, bool LOOP>
__global__ __launch_bounds__(BT) void rms_norm_bwd_kernel(BwdArgs A) {
  typedef typename El<DT>::T E;
  __shared__ float red[BT / kWave];
  constexpr int RPB = BT / T;
  __shared__ float acc_lds[RPB > 1 ? BT * kV : 1];
  const int t = threadIdx.x % T;
  const int64_t step = (int64_t)T * NV * kV;
  for (int64_t base = 0; base < (LOOP ? A.D : 1); base += step) {
    float w[NV][kV], dwa[NV][kV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t c = base + (int64_t)(i * T + t) * kV;
#pragma unroll
      for (int j = 0; j < kV; ++j) { w[i][j] = 1.0f; dwa[i][j] = 0.0f; }
      if (A.weight) load8<DT>((const E*)A.weight + c, A.D - c, A.D, w[i]);
    }
    for (int64_t blk = blockIdx.x; blk * RPB < A.R; blk += gridDim.x) {
      const int64_t row = blk * RPB + threadIdx.x / T;
      const bool on = row < A.R;
      const int64_t rr = on ? row : 0, D = on ? A.D : 0;
      const E* hp = (const E*)A.h + rr * A.ldh;
      const E* yp = (const E*)A.dy + rr * A.ldy;
      const float r = on ? A.rstd[rr] : 0.0f;
      float n[NV][kV], g[NV][kV], dot = 0.0f;
      if constexpr (LOOP) {  // the whole row's mean(g n) first
        for (int64_t b2 = 0; b2 < (A.dx ? A.D : 0); b2 += (int64_t)T * kV) {
          const int64_t c = b2 + (int64_t)t * kV;
          float a[kV], b[kV], ww[kV];
          load8<DT>(hp + c, D - c, D, a);
          load8<DT>(yp + c, D - c, D, b);
#pragma unroll
          for (int j = 0; j < kV; ++j) ww[j] = 1.0f;
          if (A.weight) load8<DT>((const E*)A.weight + c, A.D - c, A.D, ww);
#pragma unroll
          for (int j = 0; j < kV; ++j) dot = fmaf(b[j] * ww[j], a[j] * r, dot);
        }
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int64_t c = base + (int64_t)(i * T + t) * kV;
        load8<DT>(hp + c, D - c, D, n[i]);
        load8<DT>(yp + c, D - c, D, g[i]);
#pragma unroll
        for (int j = 0; j < kV; ++j) {
          n[i][j] *= r;
          dwa[i][j] = fmaf(g[i][j], n[i][j], dwa[i][j]);
          g[i][j] *= w[i][j];
          if constexpr (!LOOP) dot = fmaf(g[i][j], n[i][j], dot);
        }
      }
      if (!A.dx) continue;  // the same in every thread
      const float m = sum_row<T>(dot, red) / (float)A.D;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int64_t c = base + (int64_t)(i * T + t) * kV;
        if (c >= D) continue;
#pragma unroll
        for (int j = 0; j < kV; ++j) g[i][j] = r * fmaf(-n[i][j], m, g[i][j]);
        if (A.dh) {
          float e[kV];
          load8<DT>((const E*)A.dh + rr * A.lddh + c, D - c, D, e);
#pragma unroll
          for (int j = 0; j < kV; ++j) g[i][j] += e[j];
        }
        store8<DT>((E*)A.dx + rr * A.ldx + c, D - c, g[i]);
      }
    }
    if (!A.part) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t c = base + (int64_t)(i * T + t) * kV;
      if constexpr (RPB > 1) {  // join the workgroup's rows, in a fixed order
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kV; ++j) acc_lds[threadIdx.x * kV + j] = dwa[i][j];
        __syncthreads();
        if (threadIdx.x < T)
          for (int o = 1; o < RPB; ++o)
#pragma unroll
            for (int j = 0; j < kV; ++j) dwa[i][j] += acc_lds[(o * T + threadIdx.x) * kV + j];
      }
      if (threadIdx.x < T)
#pragma unroll
        for (int j = 0; j < kV; ++j)
          if (c + j < A.D) A.part[blockIdx.x * A.D + c + j] = dwa[i][j];
    }
  }
}

// dw[c] = sum over parts of part[p][c]: 16 columns x 16 slices of the parts a workgroup, joined in
// order.  (64 columns x 4 slices took 63 us for 1024 parts of 512 columns: 8 workgroups, 256 loads
// one after the other.)
template <int DT>
__global__ __launch_bounds__(256) void dw_sum_kernel(const float* part, int64_t parts, int64_t D, void* dw) {
  __shared__ float s[16][17];
  const int x = threadIdx.x & 15, k = threadIdx.x >> 4;
  const int64_t c = (int64_t)blockIdx.x * 16 + x;
  float a = 0.0f;
  if (c < D) {
#pragma unroll 8
    for (int64_t p = k; p < parts; p += 16) a += part[p * D + c];
  }
  s[k][x] = a;
  __syncthreads();
  if (k == 0 && c < D) {
#pragma unroll
    for (int o = 1; o < 16; ++o) a += s[o][x];
    ((typename El<DT>::T*)dw)[c] = from_f<DT>(a);
  }
}

struct QuantArgs {
  const void* x;
  uint8_t* q;
  float* scale;
  int64_t ldx, ldq, sld, R, D, xb, qb, sb;  // xb, qb, sb: strides of the batch
};

// 1 x 128 blocks: 16 lanes each, kUnits blocks one after the other (their loads in flight together)
constexpr int kUnits = 4;
template <int DT>
__global__ __launch_bounds__(256) void quant_rows_kernel(QuantArgs A) {
  typedef typename El<DT>::T E;
  const int64_t b = blockIdx.z;
  const uint32_t kb = (uint32_t)((A.D + 127) >> 7);
  const int64_t first = (int64_t)blockIdx.x * (16 * kUnits) + (threadIdx.x >> 4), row0 = first / kb;
  const uint32_t blk0 = (uint32_t)(first - row0 * kb);
  float v[kUnits][kV];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const uint32_t at = blk0 + 16 * u;
    const int64_t row = row0 + at / kb, c = (at % kb) * 128 + (threadIdx.x & 15) * kV;
    load8<DT>((const E*)A.x + b * A.xb + (row < A.R ? row : 0) * A.ldx + c, row < A.R ? A.D - c : 0, A.D, v[u]);
  }
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const uint32_t at = blk0 + 16 * u, blk = at % kb;
    const int64_t row = row0 + at / kb, c = blk * 128 + (threadIdx.x & 15) * kV;
    if (row < A.R) quant8(v[u], A.q + b * A.qb + row * A.ldq, c, A.D, A.ldq, A.scale + b * A.sb + blk * A.sld + row);
  }
}

// 128 x 128 blocks: one workgroup each, the block in registers (16 lanes a row, 16 rows a pass)
template <int DT>
__global__ __launch_bounds__(256) void quant_tiles_kernel(QuantArgs A) {
  typedef typename El<DT>::T E;
  __shared__ float red[4];
  const int64_t b = blockIdx.z, blk = blockIdx.x, rb = blockIdx.y;
  const int64_t c = blk * 128 + (threadIdx.x & 15) * kV;
  float v[8][kV], top = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = rb * 128 + i * 16 + (threadIdx.x >> 4);
    const bool on = row < A.R;
    load8<DT>((const E*)A.x + b * A.xb + (on ? row : 0) * A.ldx + c, on ? A.D - c : 0, A.D, v[i]);
#pragma unroll
    for (int j = 0; j < kV; ++j) top = fmaxf(top, fabsf(v[i][j]));
  }
  top = max_lanes<64>(top);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), kLeast);
  const Ratio inv(top);
  const int64_t pad = (A.D + 15) / 16 * 16;
  const int64_t room = (A.ldq >= pad ? pad : A.D) - c;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = rb * 128 + i * 16 + (threadIdx.x >> 4);
    if (row >= A.R || room <= 0) continue;
#pragma unroll
    for (int j = 0; j < kV; ++j) v[i][j] = inv * v[i][j];
    store8_e4m3(A.q + b * A.qb + row * A.ldq + c, A.D - c, room, pack8_e4m3(v[i]));
  }
  if (threadIdx.x == 0) A.scale[b * A.sb + blk * A.sld + rb] = top / kTop;
}

template <int DT, bool FP8>
void launch_norm(NormArgs A, hipStream_t st) {
  const int64_t D = A.D, R = A.R, e = DT == TRK_F32 ? 4 : 2;
  // at most 2^23 workgroups of 256 a launch (a launch has fewer than 2^32 threads)
  const int64_t most = ((int64_t)1 << 23) * (D <= 128 ? 16 : D <= 1024 ? 4 : 1);
  for (int64_t r = 0; r < R; r += most) {
    A.R = std::min(most, R - r);
#define TRK_NORM(T, NV, BT, LOOP) \
  rms_norm_kernel<DT, T, NV, BT, FP8, LOOP><<<(unsigned)((A.R + (BT / T) - 1) / (BT / T)), BT, 0, st>>>(A)
    if (D <= 128) TRK_NORM(16, 1, 256, false);
    else if (D <= 512) TRK_NORM(64, 1, 256, false);
    else if (D <= 1024) TRK_NORM(64, 2, 256, false);
    else if (D <= 2048) TRK_NORM(256, 1, 256, false);
    else if (D <= 4096) TRK_NORM(256, 2, 256, false);
    else if (D <= 8192) TRK_NORM(256, 4, 256, false);
    else TRK_NORM(256, 4, 256, true);
#undef TRK_NORM
    auto next = [&](auto& p, int64_t bytes) {
      if (p) p = (std::remove_reference_t<decltype(p)>)((uintptr_t)p + bytes);
    };
    next(A.x, most * A.ldx * e);
    next(A.res, most * A.ldr * e);
    next(A.y, most * A.ldy * (FP8 ? 1 : e));
    next(A.h, most * A.ldh * e);
    next(A.rstd, most * 4);
    next(A.scale, most * 4);
  }
}

// workgroups of the backward kernel, each with one partial row of dw
int64_t bwd_parts(int64_t R, int64_t D) {
  const int64_t rows = D <= 128 ? 16 : D <= 1024 ? 4 : 1;
  return std::max<int64_t>(1, std::min<int64_t>((R + rows - 1) / rows, D <= 4096 ? 1024 : 512));
}

template <int DT>
void launch_bwd(const BwdArgs& A, hipStream_t st) {
  const int64_t D = A.D;
  const unsigned grid = (unsigned)A.parts;
  // rows over more threads before more values a thread: with up to 32 values in each of 256 threads, 12800 rows
  // of 8000 took 239 us, with 8 in each of 1024 147
#define TRK_BWD(T, NV, BT, LOOP) rms_norm_bwd_kernel<DT, T, NV, BT, LOOP><<<grid, BT, 0, st>>>(A)
  if (D <= 128) TRK_BWD(16, 1, 256, false);
  else if (D <= 512) TRK_BWD(64, 1, 256, false);
  else if (D <= 1024) TRK_BWD(64, 2, 256, false);
  else if (D <= 2048) TRK_BWD(256, 1, 256, false);
  else if (D <= 4096) TRK_BWD(512, 1, 512, false);
  else if (D <= 8192) TRK_BWD(1024, 1, 1024, false);
  else if (D <= 16384) TRK_BWD(1024, 2, 1024, false);
  else TRK_BWD(1024, 2, 1024, true);
#undef TRK_BWD
  if (A.dw) dw_sum_kernel<DT><<<(unsigned)((D + 15) / 16), 256, 0, st>>>(A.part, A.parts, D, A.dw);
}

bool float_type(int dt) { return dt == TRK_F32 || dt == TRK_BF16 || dt == TRK_F16; }

#define TRK_BY_TYPE(dt, CALL)                       \
  do {                                              \
    if (dt == TRK_F32) { CALL(TRK_F32); }           \
    else if (dt == TRK_BF16) { CALL(TRK_BF16); }    \
    else { CALL(TRK_F16); }                         \
  } while (0)

int check_norm(const char* what, const void* x, int64_t ldx, const void* res, int64_t ldr, int64_t R, int64_t D,
               int dtype, const void* y, int64_t ldy, const void* h, int64_t ldh, float eps) {
  TRK_REQUIRE(float_type(dtype), "%s: dtype must be TRK_F32, TRK_BF16 or TRK_F16", what);
  TRK_REQUIRE(R >= 0 && D >= 1 && D <= (1 << 24), "%s: bad shape R=%lld D=%lld", what, (long long)R, (long long)D);
  TRK_REQUIRE(R < ((int64_t)1 << 31), "%s: R=%lld rows are too many", what, (long long)R);
  TRK_REQUIRE(eps >= 0.0f, "%s: eps must not be negative", what);
  if (R == 0) return TRK_OK;
  TRK_REQUIRE(x && y, "%s: null pointer", what);
  TRK_REQUIRE(ldx >= D && ldy >= D && (!res || ldr >= D) && (!h || ldh >= D), "%s: row stride below D", what);
  return TRK_OK;
}

}  // namespace

extern "C" {

int trk_rms_norm(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight, float eps,
                 int64_t R, int64_t D, int dtype, void* y, int64_t ldy, void* h, int64_t ldh, float* rstd,
                 void* stream) {
  if (int rc = check_norm("trk_rms_norm", x, ldx, residual, ldr, R, D, dtype, y, ldy, h, ldh, eps)) return rc;
  if (R == 0) return TRK_OK;
  const NormArgs A{x, residual, weight, y, h, rstd, nullptr, ldx, ldr, ldy, ldh, 0, R, D, eps};
  hipStream_t st = (hipStream_t)stream;
#define CALL(DT) launch_norm<DT, false>(A, st)
  TRK_BY_TYPE(dtype, CALL);
#undef CALL
  return trk::check_launch("trk_rms_norm");
}

int trk_rms_norm_fp8(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight, float eps,
                     int64_t R, int64_t D, int dtype, void* q, int64_t ldq, float* scale, int64_t scale_ld, void* h,
                     int64_t ldh, void* stream) {
  if (int rc = check_norm("trk_rms_norm_fp8", x, ldx, residual, ldr, R, D, dtype, q, ldq, h, ldh, eps)) return rc;
  if (R == 0) return TRK_OK;
  TRK_REQUIRE(scale && scale_ld >= R, "trk_rms_norm_fp8: scale [ceil(D/128)][scale_ld >= R] is required");
  const NormArgs A{x, residual, weight, q, h, nullptr, scale, ldx, ldr, ldq, ldh, scale_ld, R, D, eps};
  hipStream_t st = (hipStream_t)stream;
#define CALL(DT) launch_norm<DT, true>(A, st)
  TRK_BY_TYPE(dtype, CALL);
#undef CALL
  return trk::check_launch("trk_rms_norm_fp8");
}

int64_t trk_rms_norm_bwd_parts(int64_t R, int64_t D) { return R <= 0 || D <= 0 ? 1 : bwd_parts(R, D); }

int trk_rms_norm_bwd(const void* h, int64_t ldh, const void* weight, const float* rstd, const void* dy, int64_t ldy,
                     const void* dh, int64_t lddh, int64_t R, int64_t D, int dtype, void* dx, int64_t ldx,
                     float* part, int64_t parts, void* dw, void* stream) {
  if (int rc = check_norm("trk_rms_norm_bwd", h, ldh, dh, lddh, R, D, dtype, dy, ldy, dx, ldx, 0.0f)) return rc;
  if (!dx && !dw) return TRK_OK;
  hipStream_t st = (hipStream_t)stream;
  TRK_REQUIRE(!dw || (part && parts >= 1), "trk_rms_norm_bwd: dw needs the workspace part [parts][D]");
  if (R > 0) {
    TRK_REQUIRE(rstd, "trk_rms_norm_bwd: null pointer");
    TRK_REQUIRE(!dw || parts == bwd_parts(R, D), "trk_rms_norm_bwd: parts must be trk_rms_norm_bwd_parts(R, D)");
  }
  const BwdArgs A{h, weight, dy, dh, rstd, dx, dw, dw ? part : nullptr, ldh, ldy, lddh, ldx, R, D,
                  R > 0 ? bwd_parts(R, D) : 0};
  if (R == 0) {
    if (!dw) return TRK_OK;
#define CALL(DT) dw_sum_kernel<DT><<<(unsigned)((D + 15) / 16), 256, 0, st>>>(part, 0, D, dw)
    TRK_BY_TYPE(dtype, CALL);
#undef CALL
  } else {
#define CALL(DT) launch_bwd<DT>(A, st)
    TRK_BY_TYPE(dtype, CALL);
#undef CALL
  }
  return trk::check_launch("trk_rms_norm_bwd");
}

int trk_quantize_fp8(const void* x, int64_t ldx, int64_t xb, int64_t B, int64_t R, int64_t D, int block_rows,
                     int dtype, void* q, int64_t ldq, int64_t qb, float* scale, int64_t scale_ld, int64_t sb,
                     void* stream) {
  TRK_REQUIRE(float_type(dtype), "trk_quantize_fp8: dtype must be TRK_F32, TRK_BF16 or TRK_F16");
  TRK_REQUIRE(block_rows == 1 || block_rows == 128, "trk_quantize_fp8: block_rows must be 1 or 128");
  TRK_REQUIRE(B >= 0 && B <= 65535 && R >= 0 && D >= 1 && D <= (1 << 24) && R < ((int64_t)1 << 31),
              "trk_quantize_fp8: bad shape B=%lld R=%lld D=%lld", (long long)B, (long long)R, (long long)D);
  if (B == 0 || R == 0) return TRK_OK;
  TRK_REQUIRE(x && q && scale, "trk_quantize_fp8: null pointer");
  const int64_t kb = (D + 127) / 128, rb = block_rows == 1 ? R : (R + 127) / 128;
  TRK_REQUIRE(ldx >= D && ldq >= D && scale_ld >= rb, "trk_quantize_fp8: row stride below D, or scale_ld too small");
  const int64_t groups = block_rows == 1 ? (R * kb + 16 * kUnits - 1) / (16 * kUnits) : kb * rb;
  TRK_REQUIRE(groups * B < (1 << 24) && (block_rows == 1 || rb <= 65535), "trk_quantize_fp8: too many blocks for a launch");
  const QuantArgs A{x, (uint8_t*)q, scale, ldx, ldq, scale_ld, R, D, xb, qb, sb};
  hipStream_t st = (hipStream_t)stream;
  if (block_rows == 1) {
    const dim3 grid((unsigned)groups, 1, (unsigned)B);
#define CALL(DT) quant_rows_kernel<DT><<<grid, 256, 0, st>>>(A)
    TRK_BY_TYPE(dtype, CALL);
#undef CALL
  } else {
    const dim3 grid((unsigned)kb, (unsigned)rb, (unsigned)B);
#define CALL(DT) quant_tiles_kernel<DT><<<grid, 256, 0, st>>>(A)
    TRK_BY_TYPE(dtype, CALL);
#undef CALL
  }
  return trk::check_launch("trk_quantize_fp8");
}

}  // extern "C"
