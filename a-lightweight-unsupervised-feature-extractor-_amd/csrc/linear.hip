// Matrix products of rows and weights: 8-bit codes with an f32 scale for each block of 128
// columns, and rows sorted by group (a stream, an expert) with one weight for each group, in
// 8 or 16 bits, with the 16-bit form's two gradients.
//
//   8 bits:  y[m][n] = sum_kb sx[m][kb] sw[n][kb] (sum of the block's 128 products x w) + bias[n]
//   grouped: the counts[0] first rows by w[0], the counts[1] next by w[1], ..
//   gradients: dx = dy w[g] (row by row),  dw[g] = sum over the group's rows of dy^T x
//
// The product runs transposed on the matrix cores: w rows are the A operand and x rows the B
// operand, so a lane ends up with four consecutive columns of one row of y (one 8-byte store)
// and needs one row scale per tile.  A K step is 128 bytes of every row (one 16x16x128 e4m3 or
// two 16x16x32 16-bit matrix instructions a tile).  Which k a lane's bytes hold does not matter
// as long as both operands agree: a lane of group g = lane / 16 takes the 16-byte chunks g and
// g + 4 of its row.
#include <atomic>
#include <type_traits>

#include "trk_common.h"

using namespace trk;

namespace {

typedef float f4v __attribute__((ext_vector_type(4)));
typedef int i4v __attribute__((ext_vector_type(4)));
typedef int i8v __attribute__((ext_vector_type(8)));
typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef _Float16 h2v __attribute__((ext_vector_type(2)));

constexpr int kStep = 128;  // bytes of K a step

struct MmArgs {
  const uint8_t *x, *w;      // rows; strides below in bytes
  const float *sx, *sw, *bias;
  void* y;
  const int32_t* counts;     // grouped: rows of each group (null: one group of M rows)
  int64_t ldx, ldw, wg;      // wg: bytes from a group's weight to the next
  int64_t sx_row, sx_kb, sw_row, sw_kb, sw_g;
  int64_t ldy;               // elements
  int64_t M, N, K, G;        // K in elements
  int zero_tail;             // rows behind the last group are written as zeros
  int parts, share;          // tiles only: K in so many parts of `share` steps, each with its own y [M][N] (f32)
};

// ------------------------------------------------------------------ which rows a tile has
struct Tile {
  int64_t row0;
  int rows;   // rows of the tile; 0: none
  int g;      // group, or -1: rows behind the last group
};

// Which rows a tile (TM rows, a group's last one shorter) has, found by all BT threads from the counts:
// each thread owns a run of groups; its rows and tiles are summed and scanned once, and the thread
// whose run holds a tile walks it.  Negative counts are 0 and the sum stops at M, so no count
// reaches past the rows.
struct Runs {                 // of a thread: the first row of its groups, their first tile, how many tiles
  int first, t0, tiles;
};

template <int TM, int BT>
struct Finder {
  int live, end;             // tiles of all groups; rows of all groups
  int all;                   // tiles, with those of the rows behind the last group

  __device__ __forceinline__ static int scan(int v, int* sums, int& total) {  // exclusive, over the workgroup
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int incl = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(incl, d, 64);
      if (lane >= d) incl += o;
    }
    if (lane == 63) sums[wave] = incl;
    __syncthreads();
    int before = incl - v;
    total = 0;
#pragma unroll
    for (int w = 0; w < BT / 64; ++w) {
      if (w < wave) before += sums[w];
      total += sums[w];
    }
    __syncthreads();
    return before;
  }

  // saturating: sums of rows stop at M < 2^31 in every step
  __device__ __forceinline__ static int scan_rows(int v, int* sums, int M, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int incl = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(incl, d, 64);
      if (lane >= d) incl = (int)min((int64_t)incl + o, (int64_t)M);
    }
    const int excl = __shfl_up(incl, 1, 64);
    if (lane == 63) sums[wave] = incl;
    __syncthreads();
    int64_t before = lane > 0 ? excl : 0, all = 0;
#pragma unroll
    for (int w = 0; w < BT / 64; ++w) {
      if (w < wave) before += sums[w];
      all += sums[w];
    }
    total = (int)min(all, (int64_t)M);
    __syncthreads();
    return (int)min(before, (int64_t)M);
  }

  // groups are fewer than 2^16, rows fewer than 2^31
  __device__ void init(const int32_t* counts, int G, int64_t M, bool tail, int* sums, Runs* runs) {
    const int run = (G + BT - 1) / BT, g0 = min(G, (int)threadIdx.x * run), g1 = min(G, g0 + run);
    int64_t rows = 0;
    for (int g = g0; g < g1; ++g) rows = min(rows + max(0, counts[g]), M);
    Runs r;
    r.first = scan_rows((int)rows, sums, (int)M, end);
    r.tiles = 0;
    int64_t at = r.first;
    for (int g = g0; g < g1; ++g) {
      const int64_t c = min((int64_t)max(0, counts[g]), M - at);
      r.tiles += (int)((c + TM - 1) / TM);
      at += c;
    }
    r.t0 = scan(r.tiles, sums, live);
    runs[threadIdx.x] = r;
    all = live + (tail ? (int)((M - end + TM - 1) / TM) : 0);
  }

  // one thread writes the rows of tile t < all
  __device__ void find(const int32_t* counts, int G, int64_t M, int t, const Runs* runs, Tile* found) const {
    const Runs r = runs[threadIdx.x];
    if (t >= r.t0 && t < r.t0 + r.tiles) {
      const int run = (G + BT - 1) / BT, g0 = (int)threadIdx.x * run, g1 = min(G, g0 + run);
      int64_t at = r.first;
      int k = r.t0;
      for (int g = g0; g < g1; ++g) {
        const int64_t c = min((int64_t)max(0, counts[g]), M - at);
        const int n = (int)((c + TM - 1) / TM);
        if (t < k + n) {
          const int64_t o = (int64_t)(t - k) * TM;
          *found = Tile{at + o, (int)min((int64_t)TM, c - o), g};
          break;
        }
        k += n;
        at += c;
      }
    }
    if (threadIdx.x == 0 && t >= live) {
      const int64_t o = end + (int64_t)(t - live) * TM;
      *found = Tile{o, (int)min((int64_t)TM, M - o), -1};
    }
  }
};

// ------------------------------------------------------------------ stores of four columns
// f(integral_constant) for the output type `dt`
template <typename F>
__device__ __forceinline__ void by_type(int dt, F f) {
  if (dt == TRK_F32) f(std::integral_constant<int, TRK_F32>());
  else if (dt == TRK_BF16) f(std::integral_constant<int, TRK_BF16>());
  else f(std::integral_constant<int, TRK_F16>());
}

template <int DT>
__device__ __forceinline__ void put(void* y, int64_t at, float v) {
  if constexpr (DT == TRK_F32) ((float*)y)[at] = v;
  else if constexpr (DT == TRK_BF16) ((uint16_t*)y)[at] = f32_to_bf16(v);
  else ((_Float16*)y)[at] = (_Float16)v;
}

template <int DT>
__device__ __forceinline__ uint2 pack4(f4v v) {
  if constexpr (DT == TRK_BF16) return make_uint2(pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]));
  else
    return make_uint2(__builtin_bit_cast(uint32_t, h2v{(_Float16)v[0], (_Float16)v[1]}),
                      __builtin_bit_cast(uint32_t, h2v{(_Float16)v[2], (_Float16)v[3]}));
}

// y[at .. at + 3] (`left` of them exist); gfx950 takes the wide store at any alignment
template <int DT>
__device__ __forceinline__ void put4(void* y, int64_t at, int left, f4v v) {
  if (left >= 4) {
    if constexpr (DT == TRK_F32) {
      __builtin_memcpy((float*)y + at, &v, 16);
    } else {
      const uint2 p = pack4<DT>(v);
      __builtin_memcpy((uint16_t*)y + at, &p, 8);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (j < left) put<DT>(y, at + j, v[j]);
  }
}

// A wave's 16-byte pieces of two 64-byte runs of its 16 rows, a of columns 0 .. and b of the columns
// behind them: rows 8 .. 15 of a and 0 .. 7 of b change places, so that a holds rows 0 .. 7 of both
// runs and b rows 8 .. 15.  One store then writes 8 whole 128-byte lines and not 16 halves.
__device__ __forceinline__ void pair_lines(uint4& a, uint4& b, bool low) {
  auto turn = [&](uint32_t& u, uint32_t& v) {
    const uint32_t t = low ? v : u;  // what the other half needs
    const uint32_t r = __builtin_amdgcn_mov_dpp(t, 0x128, 0xf, 0xf, false);  // from the lane 8 further in its 16
    (low ? v : u) = r;
  };
  turn(a.x, b.x);
  turn(a.y, b.y);
  turn(a.z, b.z);
  turn(a.w, b.w);
}

constexpr int kRowsLds = 16 * 68 * 4;  // shared memory of a wave's 16 rows x 64 columns on their way out

// A wave's IT x JT tiles of 16 x 16: columns wn + 16 i + 4 lg .. + 3 of rows wm + 16 j + lr, of a tile with
// `rows` rows and `cols` columns at y (row stride ld).  bias: of the tile's columns, or null.
// 16-bit rows: lanes of odd and even lg swap halves of two neighbouring column tiles, so that a lane
// has 8 columns (16 bytes) and the pair a run of 64 bytes a row, as one tile has in 32 bits; two such
// runs are then paired to lines.
template <int IT, int JT>
__device__ __forceinline__ void store_tiles(const f4v (&acc)[IT][JT], void* y, int dt, int64_t at, int64_t ld, int rows,
                                            int cols, int wn, int wm, int lr, int lg, const float* bias, uint8_t* lds) {
  asm volatile("" : "+v"(lr), "+v"(lg));  // addresses are made here, not kept through the loops before
  by_type(dt, [&](auto t) {
    constexpr int DT = decltype(t)::value;
    typedef std::conditional_t<DT == TRK_F32, float, uint16_t> E;
    E* tile = (E*)y + at;
    auto column_bias = [&](int i) {
      f4v b = {0, 0, 0, 0};
      const int n = wn + i * 16 + lg * 4;
      if (bias)
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = n + e < cols ? bias[n + e] : 0.0f;
      return b;
    };
    // Rows that start anywhere: 64 columns of 16 rows at a time through the wave's own LDS, so that each
    // store is of one row's neighbouring columns.  2048 x 50000 x 128 to f32 (rows 64 bytes off the lines): 102 us
    // against 125 with the pieces below (92 for the whole lines of 50048 columns); 50001 columns: 107
    // against 181, in 16 bits 77 against 104.
    const bool lines = DT == TRK_F32 ? ((uintptr_t)tile | (uintptr_t)(ld * 4)) % 128 == 0
                                     : ((uintptr_t)tile | (uintptr_t)(ld * 2)) % 16 == 0;
    if (!lines) {
      constexpr int P = DT == TRK_F32 ? 68 : 72;  // elements of a row there (padded against bank conflicts)
      E* own = (E*)lds;
      const int lane = lg * 16 + lr;
#pragma unroll
      for (int h = 0; h < IT; h += 4) {
        f4v b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = column_bias(h + i);
        const int n = wn + h * 16 + lane;
#pragma unroll
        for (int j = 0; j < JT; ++j) {
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f4v v = acc[h + i][j] + b[i];
            if constexpr (DT == TRK_F32) *(f4v*)(own + lr * P + i * 16 + lg * 4) = v;
            else *(uint2*)(own + lr * P + i * 16 + lg * 4) = pack4<DT>(v);
          }
          __builtin_amdgcn_wave_barrier();  // (a wave's LDS operations keep their order)
          const int left = rows - wm - j * 16;
          if (n < cols) {
            E* to = tile + (int64_t)(wm + j * 16) * ld + n;
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (r < left) to[r * ld] = own[r * P + lane];
          }
        }
      }
    } else if (wn + IT * 16 <= cols) {  // the wave's columns are all there
      constexpr int RUN = DT == TRK_F32 ? 1 : 2;  // column tiles of a 64-byte run
      const bool low = lr < 8;
      auto run = [&](int i, int j, const f4v* b) {
        if constexpr (DT == TRK_F32) {
          return __builtin_bit_cast(uint4, acc[i][j] + b[0]);
        } else {
          typedef unsigned u2 __attribute__((ext_vector_type(2)));
          const uint2 p = pack4<DT>(acc[i][j] + b[0]), q = pack4<DT>(acc[i + 1][j] + b[1]);
          const u2 x = __builtin_amdgcn_permlane16_swap(p.x, q.x, false, false);
          const u2 z = __builtin_amdgcn_permlane16_swap(p.y, q.y, false, false);
          return make_uint4(x[0], z[0], x[1], z[1]);
        }
      };
      // a lane's column in a run; lanes of the upper rows hold the second run
      const int n = wn + (DT == TRK_F32 ? lg * 4 : (lg & 1) * 16 + (lg >> 1) * 8) + (low ? 0 : RUN * 16);
#pragma unroll
      for (int i = 0; i < IT; i += 2 * RUN) {
        f4v b[2 * RUN];
#pragma unroll
        for (int h = 0; h < 2 * RUN; ++h) b[h] = column_bias(i + h);
#pragma unroll
        for (int j = 0; j < JT; ++j) {
          uint4 u = run(i, j, b), v = run(i + RUN, j, b + RUN);
          pair_lines(u, v, low);
          const int m = wm + j * 16 + (lr & 7);
          E* to = tile + m * ld + n + i * 16;
          if (m < rows) __builtin_memcpy(to, &u, 16);
          if (m + 8 < rows) __builtin_memcpy(to + 8 * ld, &v, 16);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int n = wn + i * 16 + lg * 4;
        if (n >= cols) continue;
        const f4v b = column_bias(i);
#pragma unroll
        for (int j = 0; j < JT; ++j) {
          const int m = wm + j * 16 + lr;
          if (m < rows) put4<DT>(tile, m * ld + n, cols - n, acc[i][j] + b);
        }
      }
    }
  });
}

// ------------------------------------------------------------------ one K step of one tile
enum { IN_E4M3 = 0, IN_BF16 = 1, IN_F16 = 2, IN_E4M3X = 3 };

constexpr bool is8(int in) { return in == IN_E4M3 || in == IN_E4M3X; }

// A lane's 32 bytes of a row's K step, as the matrix instruction takes them.  IN_E4M3 is the 8-bit
// instruction: in each 8 bytes it cuts every product, towards zero, by less than 2^-13 of the largest one (to multiples
// of 2^-13 of the power of two that the largest one's exponents add up to; measured: 256 * 256 - 256 * 256 + s * 1
// leaves the multiple of 8 below s in the same 8 columns, s in any others; 1.5e-5 of an ordinary sum in the root
// mean square).  That is far below half a step of a 16-bit y unless products cancel, so 16-bit outputs use it, and the interface says so.  IN_E4M3X,
// for f32 outputs, widens the codes to bf16 (exact) and multiplies at half the rate with f32 sums.
template <int IN> struct Frag {
  uint4 v[2];
  __device__ __forceinline__ void set(uint4 a, uint4 b) { v[0] = a; v[1] = b; }
};
template <> struct Frag<IN_E4M3X> {
  b8v v[4];
  __device__ __forceinline__ void set(uint4 a, uint4 b) {
    const uint32_t t[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      typedef __bf16 b2v __attribute__((ext_vector_type(2)));
      const b2v p0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(t[2 * q], 1.0f, false);
      const b2v p1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(t[2 * q], 1.0f, true);
      const b2v p2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(t[2 * q + 1], 1.0f, false);
      const b2v p3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(t[2 * q + 1], 1.0f, true);
      v[q] = b8v{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
    }
  }
};

template <int IN>
__device__ __forceinline__ f4v mma(const Frag<IN>& a, const Frag<IN>& b, f4v c) {
  if constexpr (IN == IN_E4M3) {
    const i8v x = {(int)a.v[0].x, (int)a.v[0].y, (int)a.v[0].z, (int)a.v[0].w,
                   (int)a.v[1].x, (int)a.v[1].y, (int)a.v[1].z, (int)a.v[1].w};
    const i8v y = {(int)b.v[0].x, (int)b.v[0].y, (int)b.v[0].z, (int)b.v[0].w,
                   (int)b.v[1].x, (int)b.v[1].y, (int)b.v[1].z, (int)b.v[1].w};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 0, 0, 0, 0, 0, 0);
  } else if constexpr (IN == IN_E4M3X) {
#pragma unroll
    for (int q = 0; q < 4; ++q) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[q], b.v[q], c, 0, 0, 0);
    return c;
  } else {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      if constexpr (IN == IN_BF16)
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8v, a.v[q]), __builtin_bit_cast(b8v, b.v[q]), c,
                                                    0, 0, 0);
      else
        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8v, a.v[q]), __builtin_bit_cast(h8v, b.v[q]), c,
                                                   0, 0, 0);
    }
    return c;
  }
}

// LDS tile of rows of 128 bytes; a row's 16-byte chunks are rotated by XOR with the row so that
// eight rows' reads of one chunk fall into different banks
__device__ __forceinline__ int lds_at(int row, int chunk) { return row * kStep + ((chunk ^ (row & 7)) << 4); }

template <int IN>
__device__ __forceinline__ Frag<IN> frag(const uint8_t* tile, int row, int lg) {
  Frag<IN> f;
  f.set(*(const uint4*)(tile + lds_at(row, lg)), *(const uint4*)(tile + lds_at(row, lg + 4)));
  return f;
}

// 16 bytes at p, of which `left` exist (the rest 0), in a row of `row` bytes that ends with them: a part
// piece is the row's last 16 bytes, shifted down
__device__ __forceinline__ uint4 load16(const uint8_t* p, int64_t left, int64_t row) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (left >= 16) {
    __builtin_memcpy(&v, p, 16);
  } else if (left > 0 && row >= 16) {
    const int s = 16 - (int)left;
    uint64_t t[2];
    __builtin_memcpy(t, p - s, 16);
    if (s >= 8) {
      t[0] = t[1] >> (8 * (s - 8));
      t[1] = 0;
    } else {
      t[0] = t[0] >> (8 * s) | t[1] << (64 - 8 * s);
      t[1] >>= 8 * s;
    }
    __builtin_memcpy(&v, t, 16);
  } else if (left > 0) {
    uint8_t t[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) t[j] = j < left ? p[j] : 0;
    __builtin_memcpy(&v, t, 16);
  }
  return v;
}

// ------------------------------------------------------------------ large tiles
#define GPTR(p) ((const __attribute__((address_space(1))) void*)(p))
#define LPTR(p) ((__attribute__((address_space(3))) void*)(p))

// 16 bytes a lane from base + voff + soff to LDS (lane l of the wave at lds + 16 l)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_at(const uint8_t* base, int64_t bytes) {
  const uint64_t u = reinterpret_cast<uint64_t>(base);  // the same in every lane
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u), hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
  const uint32_t n = __builtin_amdgcn_readfirstlane((uint32_t)min(bytes, (int64_t)0xffffffff));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>((uint64_t)hi << 32 | lo), 0, n, 0x00020000);
}
__device__ __forceinline__ void to_lds(__amdgpu_buffer_rsrc_t r, uint8_t* lds, uint32_t voff, uint32_t soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, LPTR(lds), 16, voff, soff, 0, 0);
}

// work item `id` of `n` on the XCD that runs it (workgroup id % 8): each XCD gets a contiguous run
__device__ __forceinline__ int64_t xcd_run(int64_t id, int64_t n) {
  const int64_t per = n / 8, more = n % 8, x = id % 8;
  return x * per + min(x, more) + id / 8;
}

// The product.  Bound by the matrix cores at the clock the chip holds under them: 8192 x 8192 x 8192 in 8 bits
// 465 us (455-480 over 100 traced launches; 2.4 PFLOP/s; the library's product with one scale for all runs at 2.7,
// 408 us), matrix instructions busy 59 % of the cycles at 1.9 GHz; in 16 bits 835 us (1.3 PFLOP/s, the library
// 813); in 8 bits to f32, with 128-tiles at half the rate, 950.  Few steps a tile leave more to the first copies and
// stores: 64 ragged groups, 65536 x 2048 x 1024 in 8 bits 232 us, matrix instructions busy 29 %; 16 of 16384 x
// 2048 x 2048 in 16 bits 179 us, 35 %.  What brought the 8-bit
// one there, us: 128-tiles through registers 2064, 256-tiles with straight copies a step ahead 547, copies
// spread over the step 484, several tiles a workgroup 478, rows of tiles kept in order 424-457.  Tried and
// dropped: 128 x 256 and 256 x 128 tiles with two or three stages (562-650 us; more bytes to LDS for each
// operation), four waves of 128 x 128 (949: one wave a SIMD hides nothing), workgroups that start apart and
// stores that stay in flight into the next tile's first step (no change: a wave is held while its
// stores are taken in, so a tile of few steps pays for them, about 6 us of 22 at 256 x 256 x 1024).
//
// TN x TM tiles, WN x WM waves, operands copied to LDS one step ahead.  DMA: straight, 16 bytes a lane;
// every row starts at a multiple of 16 bytes.  Else through registers, at any alignment.  A
// workgroup runs several tiles: the next tile's first copies are sent before a tile's stores.
template <int IN, bool WROW, bool DMA, int TN, int TM, int WN, int WM>
__global__ __launch_bounds__(WN * WM * 64, 2) void mm_tile_kernel(MmArgs A, int dt, int ntiles, int mtiles) {
  constexpr int BT = WN * WM * 64, IT = TN / WN / 16, JT = TM / WM / 16;
  constexpr int XB = TM * kStep, WB = TN * kStep, LS = is8(IN) ? (TM + TN + BT - 1) / BT : 0, STAGE = XB + WB + LS * BT * 4;
  constexpr int LX = TM * 8 / BT, LW = TN * 8 / BT, LOADS = LX + LW + LS, PER = (LOADS + IT - 1) / IT;
  static_assert(TM * 8 % BT == 0 && TN * 8 % BT == 0 && TM % 64 == 0, "whole loads");
  static_assert(WROW || 128 % (TN / WN) == 0, "a wave's columns lie in one block of 128");
  static_assert(WN * WM * kRowsLds <= STAGE && IT % 4 == 0, "stores go through one stage");
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  __shared__ int sums[BT / 64];
  __shared__ Runs runs[BT];
  __shared__ Tile found[2];  // of this tile and the next, in turn: a wave may be a barrier ahead
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = (wave % WN) * (TN / WN), wm = (wave / WN) * (TM / WM), lr = lane & 15, lg = lane >> 4;
  Finder<TM, BT> F;
  if (A.counts) {
    F.init(A.counts, (int)A.G, A.M, A.zero_tail, sums, runs);
    mtiles = __builtin_amdgcn_readfirstlane(F.all);
  }
  const int64_t total = (int64_t)ntiles * mtiles * A.parts;

  // the tile that is worked on: its rows, columns and sources
  int64_t row0, n0;
  int rows, cols, grp, steps, rest, part;
  int64_t kbytes;
  const uint8_t *xb, *wb;
  uint32_t x0, w0, xend, wend;  // a lane's first piece of its operand's rows, and its piece of the last row
  const float* ssrc[LS > 0 ? LS : 1];
  int next_part = 0;
  auto tile_at = [&](int64_t idx, int& nt, int& mt) {
    // bands of 8 column tiles, row tiles inside a band one after the other: an XCD's share of the
    // grid at any time is near square, so its L2 serves most operand reads
    int id = (int)xcd_run(idx, total);
    next_part = id % A.parts;
    id /= A.parts;
    const int bsize = 8 * mtiles, band = id / bsize, in = id - band * bsize;
    const int width = min(8, ntiles - band * 8);
    nt = band * 8 + in % width;
    mt = in / width;
  };
  auto setup = [&](int nt, int mt, const Tile& found) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // (as in store_tiles)
    if (A.counts) {
      row0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)found.row0);  // rows are below 2^31
      rows = __builtin_amdgcn_readfirstlane(found.rows);
      grp = __builtin_amdgcn_readfirstlane(found.g);
    } else {
      row0 = (int64_t)mt * TM;
      rows = (int)min((int64_t)TM, A.M - row0);
      grp = 0;
    }
    n0 = (int64_t)nt * TN;
    cols = (int)min((int64_t)TN, A.N - n0);
    part = next_part;
    const int64_t k0 = (int64_t)part * A.share * kStep;  // (0 where K is whole)
    kbytes = grp < 0 ? 0 : A.K * (is8(IN) ? 1 : 2) - k0;  // (no part is empty)
    if (A.parts > 1) kbytes = min(kbytes, (int64_t)A.share * kStep);
    steps = (int)(kbytes / kStep);
    rest = steps * kStep < kbytes;  // a last, partial step: masked loads through registers
    const int64_t g = max(0, grp);
    xb = A.x + row0 * A.ldx + k0;
    wb = A.w + g * A.wg + n0 * A.ldw + k0;
    // LDS slot p of an operand holds row p / 8, chunk (p % 8) ^ (row % 8): a lane's q-th copy is of row
    // tid / 8 + q BT / 8; rows past the end repeat the last one
    const uint32_t c = ((tid & 7) ^ ((tid >> 3) & 7)) << 4;
    x0 = (uint32_t)(tid >> 3) * (uint32_t)A.ldx + c;
    w0 = (uint32_t)(tid >> 3) * (uint32_t)A.ldw + c;
    xend = (uint32_t)(rows - 1) * (uint32_t)A.ldx + c;
    wend = (uint32_t)(cols - 1) * (uint32_t)A.ldw + c;
#pragma unroll
    for (int q = 0; q < LS; ++q) {  // scales: TM of the rows, then TN of the columns (whole waves of each)
      const int p = q * BT + tid, r = p - TM;
      ssrc[q] = p < TM ? A.sx + (row0 + min(p, rows - 1)) * A.sx_row
                       : A.sw + g * A.sw_g + (WROW ? n0 + min(r, cols - 1) : (n0 + min(r, cols - 1)) / 128) * A.sw_row;
      ssrc[q] += (p < TM ? A.sx_kb : A.sw_kb) * (int64_t)part * A.share;
    }
  };
  auto xoff = [&](int q) { return min(x0 + (uint32_t)(q * (BT / 8)) * (uint32_t)A.ldx, xend); };
  auto woff = [&](int q) { return min(w0 + (uint32_t)(q * (BT / 8)) * (uint32_t)A.ldw, wend); };
  // copy q of LOADS of step kt into its stage; without DMA, into `hold`, which keep() writes there
  typedef __amdgpu_buffer_rsrc_t Rsrc;
  auto copy = [&](int q, int kt, uint8_t* d, Rsrc xr, Rsrc wr, uint4* hold) __attribute__((always_inline)) {
    if (q < LX) {
      if constexpr (DMA) to_lds(xr, d + (q * BT + wave * 64) * 16, xoff(q), kt * kStep);
      else __builtin_memcpy(hold + q, xb + xoff(q) + (int64_t)kt * kStep, 16);
    } else if (q < LX + LW) {
      if constexpr (DMA) to_lds(wr, d + XB + ((q - LX) * BT + wave * 64) * 16, woff(q - LX), kt * kStep);
      else __builtin_memcpy(hold + q, wb + woff(q - LX) + (int64_t)kt * kStep, 16);
    } else {
      const int p = q - LX - LW;
      const int64_t kb = (p * BT + wave * 64 < TM ? A.sx_kb : A.sw_kb) * (int64_t)kt;
      __builtin_amdgcn_global_load_lds(GPTR(ssrc[p] + kb), LPTR(d + XB + WB + (p * BT + wave * 64) * 4), 4, 0, 0);
    }
  };
  auto keep = [&](uint8_t* d, const uint4* hold) __attribute__((always_inline)) {
    if constexpr (!DMA) {
#pragma unroll
      for (int q = 0; q < LX + LW; ++q) *(uint4*)(d + (q * BT + tid) * 16) = hold[q];  // (XB is LX BT 16)
    }
  };

  f4v acc[IT][JT];
  // One step of stage `st`; the copies go into `nx` (a different stage, so that the compiler lets
  // them stay in flight across the reads).  8 bits: the scaling of one row of tiles runs on the
  // vector units under the matrix instructions of the next.
  auto step = [&](auto more, const uint8_t* __restrict st, uint8_t* __restrict nx, int kn, Rsrc xr, Rsrc wr)
      __attribute__((always_inline)) {
    const uint8_t *xs = st, *ws = st + XB;
    const float* ss = (const float*)(st + XB + WB);
    Frag<IN> b[JT], a[2];
    float s[JT];
    f4v p[2][JT], sc[2];
    uint4 hold[LX + LW];
#pragma unroll
    for (int j = 0; j < JT; ++j) b[j] = frag<IN>(xs, wm + j * 16 + lr, lg);
    a[0] = frag<IN>(ws, wn + lr, lg);
    if constexpr (is8(IN)) {
#pragma unroll
      for (int j = 0; j < JT; ++j) {
        s[j] = ss[wm + j * 16 + lr];
        if constexpr (!WROW) s[j] *= ss[TM + wn];  // a wave's columns lie in one block of 128
      }
      if constexpr (WROW) sc[0] = *(const f4v*)(ss + TM + wn + lg * 4);
    }
    auto add = [&](int i) {
      if constexpr (is8(IN)) {
#pragma unroll
        for (int j = 0; j < JT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[i][j][e] = fmaf(p[i & 1][j][e], WROW ? s[j] * sc[i & 1][e] : s[j], acc[i][j][e]);
      }
    };
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      if (i + 1 < IT) a[(i + 1) & 1] = frag<IN>(ws, wn + (i + 1) * 16 + lr, lg);
#pragma unroll
      for (int j = 0; j < JT; ++j) {
        if constexpr (is8(IN)) p[i & 1][j] = mma<IN>(a[i & 1], b[j], f4v{0, 0, 0, 0});
        else acc[i][j] = mma<IN>(a[i & 1], b[j], acc[i][j]);
      }
      if (i > 0) add(i - 1);
      // the next step's copies, a share with each row of tiles: sent all at once they hold up the
      // wave's first reads while the memory pipe is full
      if constexpr (decltype(more)::value) {
#pragma unroll
        for (int q = i * PER; q < (i + 1) * PER; ++q)
          if (q < LOADS) copy(q, kn, nx, xr, wr, hold);
      }
      if constexpr (is8(IN) && WROW) {
        if (i + 1 < IT) sc[(i + 1) & 1] = *(const f4v*)(ss + TM + wn + (i + 1) * 16 + lg * 4);
      }
      if constexpr (is8(IN)) {
        // order of this part: the next row's reads, then a matrix instruction and the four operations
        // (eight with scales by column) of the tile before it, in turn
        __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
#pragma unroll
        for (int j = 0; j < JT; ++j) {
          __builtin_amdgcn_sched_group_barrier(0x008, IN == IN_E4M3 ? 1 : 4, 0);
          __builtin_amdgcn_sched_group_barrier(0x002, WROW ? 8 : 4, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x010, PER, 0);
      }
      __builtin_amdgcn_sched_barrier(0);  // rows of tiles stay in this order
    }
    add(IT - 1);
    if constexpr (decltype(more)::value) keep(nx, hold);
  };
  auto first_copies = [&](uint8_t* __restrict st) __attribute__((always_inline)) {
    if (steps == 0) return;
    const Rsrc xr = rows_at(xb, (rows - 1) * A.ldx + kbytes), wr = rows_at(wb, (cols - 1) * A.ldw + kbytes);
    uint4 hold[LX + LW];
#pragma unroll
    for (int q = 0; q < LOADS; ++q) copy(q, 0, st, xr, wr, hold);
    keep(st, hold);
  };

  int64_t idx = blockIdx.x;
  if (idx >= total) return;
  int nt, mt, at = 0;  // at: the stage of the step, 0 or 1
  tile_at(idx, nt, mt);
  if (A.counts) {
    F.find(A.counts, (int)A.G, A.M, mt, runs, found);
    __syncthreads();
  }
  setup(nt, mt, found[0]);
  first_copies(smem);
  for (int turn = 1;; turn ^= 1) {
    {
      const Rsrc xr = rows_at(xb, (rows - 1) * A.ldx + kbytes), wr = rows_at(wb, (cols - 1) * A.ldw + kbytes);
#pragma unroll
      for (int i = 0; i < IT; ++i)
#pragma unroll
        for (int j = 0; j < JT; ++j) acc[i][j] = f4v{0, 0, 0, 0};
      for (int kt = 0; kt < steps - 1; ++kt) {
        // step kt has landed, and every wave is done with step kt - 1, whose stage the next copies overwrite
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        step(std::true_type(), smem + at * STAGE, smem + (at ^ 1) * STAGE, kt + 1, xr, wr);
        at ^= 1;
      }
      for (int kt = max(0, steps - 1); kt < steps + rest; ++kt) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (kt == steps) {
          int t = tid;
          asm volatile("" : "+v"(t));  // (as in store_tiles)
          const int64_t k = (int64_t)steps * kStep;
          uint8_t* d = smem + at * STAGE;
#pragma unroll
          for (int q = 0; q < LX; ++q) {
            const int p = q * BT + t, c = (p & 7) ^ ((p >> 3) & 7);
            *(uint4*)(d + p * 16) = load16(xb + xoff(q) + k, kbytes - k - c * 16, kbytes);
          }
#pragma unroll
          for (int q = 0; q < LW; ++q) {
            const int p = q * BT + t, c = (p & 7) ^ ((p >> 3) & 7);
            *(uint4*)(d + XB + p * 16) = load16(wb + woff(q) + k, kbytes - k - c * 16, kbytes);
          }
#pragma unroll
          for (int q = 0; q < LS; ++q) {
            const int p = q * BT + t;
            *(float*)(d + XB + WB + p * 4) = ssrc[q][(p < TM ? A.sx_kb : A.sw_kb) * steps];
          }
          __syncthreads();
        }
        step(std::false_type(), smem + at * STAGE, smem, 0, xr, wr);
        at ^= 1;
      }
    }
    // the tile's end: its stores, through the stage `free` where rows do not suit, behind the next one's copies
    const int64_t y0 = (part * A.M + row0) * A.ldy + n0;
    const float* bias = A.bias && grp >= 0 ? A.bias + n0 : nullptr;
    const int yrows = rows, ycols = cols;
    idx += gridDim.x;
    const bool more = idx < total;
    if (more) {
      tile_at(idx, nt, mt);
      if (A.counts) F.find(A.counts, (int)A.G, A.M, mt, runs, found + turn);
    }
    // every wave is done with the last step's stage (and `found` is written)
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    auto finish = [&](uint8_t* __restrict st, uint8_t* __restrict free) __attribute__((always_inline)) {
      if (more) {
        setup(nt, mt, found[turn]);
        first_copies(st);
      }
      store_tiles(acc, A.y, dt, y0, A.ldy, yrows, ycols, wn, wm, lr, lg, bias, free + wave * kRowsLds);
    };
    finish(smem + at * STAGE, smem + (at ^ 1) * STAGE);
    if (!more) break;
  }
}

// y = sum over the parts, in order, + bias; four columns a thread.  Grouped: the rows behind the last group, which
// have no parts, are zeros (zero_tail) or stay as they are.
__global__ __launch_bounds__(256) void mm_join_kernel(MmArgs A, const float* part, int dt) {
  __shared__ int64_t sums[4];
  const float* bias = A.bias;
  const int64_t M = A.M, N = A.N, n4 = (N + 3) / 4;
  int64_t end = M;
  if (A.counts) {  // fewer than 2^16 counts below 2^31
    int64_t rows = 0;
    for (int64_t g = threadIdx.x; g < A.G; g += 256) rows += max(0, A.counts[g]);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) rows += __shfl_xor(rows, d, 64);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = rows;
    __syncthreads();
    end = min(M, sums[0] + sums[1] + sums[2] + sums[3]);
  }
  const int64_t rows = A.zero_tail ? M : end;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * n4; i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / n4, n = (i - m * n4) * 4;
    const int left = (int)min((int64_t)4, N - n);
    f4v a = {0, 0, 0, 0};
    for (int64_t p = 0; p < (m < end ? A.parts : 0); ++p) {
      const float* q = part + (p * M + m) * N + n;
      f4v v = {0, 0, 0, 0};
      if (left == 4) __builtin_memcpy(&v, q, 16);
      else
        for (int e = 0; e < left; ++e) v[e] = q[e];
      a += v;
    }
    if (bias)
      for (int e = 0; e < left; ++e) a[e] += bias[n + e];
    by_type(dt, [&](auto t) { put4<decltype(t)::value>(A.y, m * A.ldy + n, left, a); });
  }
}

// ------------------------------------------------------------------ few rows
// 16 JT rows by 16 columns a wave, the operands straight from memory to registers: with few rows the
// weights are read once and that is what counts (16 x 4096 x 4096 in 8 bits 7.2 us, 2.4 TB/s: one round of latencies;
// 16 x 8192 x 8192 20 us, 3.4 TB/s).
// KW waves of the 8 share 16 columns, each with every KW-th step, and are joined in order through
// LDS; the others take the next columns.  U steps are loaded before they are multiplied.  Any
// alignment.
template <int IN, bool WROW, int JT, int KW>
__global__ __launch_bounds__(512) void mm_few_kernel(MmArgs A, int dt) {
  constexpr int TM = 16 * JT, NW = 8 / KW, U = JT >= 4 || IN == IN_E4M3X ? 2 : 4;
  __shared__ f4v part[8][JT][64];
  __shared__ int sums[8];
  __shared__ Runs runs[512];
  __shared__ Tile found;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 15, lg = lane >> 4, kw = wave % KW;
  const int64_t n0 = ((int64_t)blockIdx.x * NW + wave / KW) * 16;
  int64_t row0 = (int64_t)blockIdx.y * TM;
  int rows, g = 0;
  if (A.counts) {
    Finder<TM, 512> F;
    F.init(A.counts, (int)A.G, A.M, A.zero_tail, sums, runs);
    if (blockIdx.y >= F.all) return;
    F.find(A.counts, (int)A.G, A.M, blockIdx.y, runs, &found);
    __syncthreads();
    row0 = found.row0;
    rows = __builtin_amdgcn_readfirstlane(found.rows);
    g = __builtin_amdgcn_readfirstlane(found.g);
  } else {
    rows = (int)min((int64_t)TM, A.M - row0);
  }
  const int cols = (int)min((int64_t)16, A.N - n0);  // may be <= 0: this wave only takes part in the barrier
  const int64_t kbytes = g < 0 ? 0 : A.K * (is8(IN) ? 1 : 2);
  const int steps = (int)((kbytes + kStep - 1) / kStep);
  f4v acc[JT];
#pragma unroll
  for (int j = 0; j < JT; ++j) acc[j] = f4v{0, 0, 0, 0};
  if (cols > 0) {
    const int64_t gw = max(0, g);
    const uint8_t* wp = A.w + gw * A.wg + (n0 + min(lr, cols - 1)) * A.ldw + lg * 16;
    const uint8_t* xp[JT];
    const float* sx[JT];
#pragma unroll
    for (int j = 0; j < JT; ++j) {
      const int64_t r = row0 + min(j * 16 + lr, rows - 1);
      xp[j] = A.x + r * A.ldx + lg * 16;
      sx[j] = A.sx + r * A.sx_row;
    }
    const float* sw = A.sw + gw * A.sw_g;
    const float* swr[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) swr[e] = sw + (WROW ? n0 + min(lg * 4 + e, cols - 1) : n0 / 128) * A.sw_row;
    for (int k0 = kw; k0 < steps; k0 += KW * U) {
      uint4 a[U][2], b[U][JT][2];
      float s[U][JT], w[U][WROW ? 4 : 1];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int kt = k0 + u * KW;
        if (kt >= steps) break;
        const int64_t k = (int64_t)kt * kStep, left = kbytes - k - lg * 16;
        if (k + kStep <= kbytes) {  // the same in every lane
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            __builtin_memcpy(&a[u][h], wp + k + h * 64, 16);
#pragma unroll
            for (int j = 0; j < JT; ++j) __builtin_memcpy(&b[u][j][h], xp[j] + k + h * 64, 16);
          }
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            a[u][h] = load16(wp + k + h * 64, left - h * 64, kbytes);
#pragma unroll
            for (int j = 0; j < JT; ++j) b[u][j][h] = load16(xp[j] + k + h * 64, left - h * 64, kbytes);
          }
        }
        if constexpr (is8(IN)) {
#pragma unroll
          for (int j = 0; j < JT; ++j) s[u][j] = sx[j][kt * A.sx_kb];
        }
        if constexpr (is8(IN)) {
#pragma unroll
          for (int e = 0; e < (WROW ? 4 : 1); ++e) w[u][e] = swr[e][kt * A.sw_kb];
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (k0 + u * KW >= steps) break;
        Frag<IN> fa;
        fa.set(a[u][0], a[u][1]);
#pragma unroll
        for (int j = 0; j < JT; ++j) {
          Frag<IN> fb;
          fb.set(b[u][j][0], b[u][j][1]);
          if constexpr (is8(IN)) {
            const f4v p = mma<IN>(fa, fb, f4v{0, 0, 0, 0});
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[j][e] = fmaf(p[e], s[u][j] * w[u][WROW ? e : 0], acc[j][e]);
          } else {
            acc[j] = mma<IN>(fa, fb, acc[j]);
          }
        }
      }
    }
  }
  if constexpr (KW > 1) {
    if (kw > 0)
#pragma unroll
      for (int j = 0; j < JT; ++j) part[wave][j][lane] = acc[j];
    __syncthreads();
    if (kw > 0) return;
#pragma unroll
    for (int o = 1; o < KW; ++o)
#pragma unroll
      for (int j = 0; j < JT; ++j) acc[j] += part[wave + o][j][lane];
  }
  const int n = lg * 4;
  if (n >= cols) return;
  f4v bias = {0, 0, 0, 0};
  if (A.bias && g >= 0)
#pragma unroll
    for (int e = 0; e < 4; ++e) bias[e] = n + e < cols ? A.bias[n0 + n + e] : 0.0f;
  by_type(dt, [&](auto t) {
#pragma unroll
    for (int j = 0; j < JT; ++j) {
      const int m = j * 16 + lr;
      if (m < rows) put4<decltype(t)::value>(A.y, (row0 + m) * A.ldy + n0 + n, cols - n, acc[j] + bias);
    }
  });
}

// ------------------------------------------------------------------ gradients (16 bits)
struct GradArgs {
  const uint16_t *dy, *x, *w;
  void *dx, *dw;                                   // null: not wanted
  const int32_t* counts;
  int64_t ldy, ldx, ldw, wg, lddx, ldo, og;        // elements; ldo, og: rows and groups of dw
  int64_t M, N, K, G;
  float* part;                                     // [parts][G][N][K]: dw in parts of each group's rows
  int64_t parts;
};

typedef short s4v __attribute__((ext_vector_type(4)));

// A turned tile keeps its source's order, [64 k][T cols], and is turned while it is read: for 16
// lanes that name 4 rows x 16 columns (4 lanes of 8 bytes a row) the transposing read returns to
// lane i the four rows' values of column i.  32-byte pieces of a row are rotated by XOR with
// the row, so that the 16 rows a wave's read touches spread over the banks.
__device__ __forceinline__ int turn_of(int row) { return (row & 3) | ((row >> 1) & 4); }

// byte of a turned tile that a lane reads for the 16 columns from col0 on (a multiple of 16) and rows 0 .. 3;
// the other columns of a wave are at this XOR 32 i, the other rows at constant distances
template <int T>
__device__ __forceinline__ uint32_t turned_at(int col0, int lane) {
  const int j = lane & 15, row = 8 * (lane >> 4) + (j >> 2);
  return row * (T * 2) + (((col0 >> 4) ^ turn_of(row)) << 5) + (j & 3) * 8;
}

template <int IN, int T>
__device__ __forceinline__ Frag<IN> frag_turned(const uint8_t* tile, uint32_t at) {
  uint2 h[4];
#pragma unroll
  for (int q = 0; q < 4; ++q)
    h[q] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v*)(
                                         tile + at + (32 * (q >> 1) + 4 * (q & 1)) * T * 2)));
  Frag<IN> f;
  f.set(make_uint4(h[0].x, h[0].y, h[1].x, h[1].y), make_uint4(h[2].x, h[2].y, h[3].x, h[3].y));
  return f;
}

// The gradients: 16 groups of 16384 rows in all, 2048 x 2048: both in 320 us (314-324 over 100 traced launches;
// 860 TFLOP/s, matrix instructions busy 40 % of the cycles; 2000 us through registers with scalar turns, 390 in two
// launches).  The last round of tiles and each tile's first copies and stores cost what is missing to the
// product's rate.
//
// T x T tile `block` of dx (DW false: rows m of one group, columns k, contracted over n) or of dw[g] (rows n,
// columns k, contracted over the group's rows), 8 waves, copies one step of 64 ahead.
template <int IN, bool DW, bool DMA>
__device__ __forceinline__ void grad_tile(const GradArgs& A, int dt, int64_t block, int64_t ctiles, int64_t rtiles, uint8_t* smem,
                                          int* sums, Runs* runs, Tile* found) {
  constexpr int T = 256, BT = 512, WN = 2, WM = 4, IT = T / WN / 16, JT = T / WM / 16;
  constexpr int XB = T * kStep, STAGE = 2 * XB, L = T * 8 / BT;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 15, lg = lane >> 4, wn = (wave % WN) * (T / WN), wm = (wave / WN) * (T / WM);
  Finder<T, BT> F;
  if constexpr (!DW) {
    F.init(A.counts, (int)A.G, A.M, true, sums, runs);
    rtiles = F.all;
  }
  const int64_t total = ctiles * rtiles * (DW ? A.G * A.parts : 1);
  if (block >= total) return;
  // dx: a contiguous run of tiles for each XCD.  dw: a run of every group's tiles for each XCD, because
  // groups differ in length (runs over the groups: dw alone 267 us against 211 for 16 groups of 16384 rows)
  int64_t id = block;
  if constexpr (DW) {
    const int64_t each = ctiles * rtiles;
    if (each % 8 == 0) id = id / each * each + xcd_run(id % each, each);
  } else {
    id = xcd_run(id, total);
  }
  const int64_t ct = id % ctiles, rt = id / ctiles;
  const int64_t c0 = ct * T;
  const int cols = (int)min((int64_t)T, A.K - c0);
  int64_t row0, steps_of;  // first output row; length of the contraction
  int rows;
  const uint16_t *wsrc0, *xsrc0;
  int64_t wld, xld;
  void* out = DW ? A.dw : A.dx;
  int64_t ldo = DW ? A.ldo : A.lddx, out0 = 0;
  if constexpr (DW) {
    const int64_t gs = rt / rtiles, g = gs / A.parts, part = gs % A.parts;
    int64_t before = 0;
    for (int64_t i = tid; i < g; i += BT) before = min(before + max(0, A.counts[i]), A.M);
    int end;
    Finder<T, BT>::scan_rows((int)before, sums, (int)A.M, end);
    int64_t first = end;
    steps_of = min((int64_t)max(0, A.counts[g]), A.M - first);
    if (A.parts > 1) {  // this part's share of the rows, in whole steps
      const int64_t share = ((steps_of + 63) / 64 + A.parts - 1) / A.parts * 64, skip = min(part * share, steps_of);
      first += skip;
      steps_of = min(share, steps_of - skip);
      out = A.part + (part * A.G + g) * A.N * A.K;
      ldo = A.K;
      dt = TRK_F32;
    } else {
      out0 = g * A.og;
    }
    row0 = (rt % rtiles) * T;
    rows = (int)min((int64_t)T, A.N - row0);
    wsrc0 = A.x + first * A.ldx + c0;
    wld = A.ldx;
    xsrc0 = A.dy + first * A.ldy + row0;
    xld = A.ldy;
  } else {
    F.find(A.counts, (int)A.G, A.M, (int)rt, runs, found);
    __syncthreads();
    const Tile t = *found;
    row0 = t.row0;
    rows = t.rows;
    steps_of = t.g < 0 ? 0 : A.N;
    wsrc0 = A.w + max(0, t.g) * A.wg + c0;
    wld = A.ldw;
    xsrc0 = A.dy + row0 * A.ldy;
    xld = A.ldy;
  }
  const int steps = (int)(steps_of / 64);
  // turned: slot p holds 8 values of row p / 32; columns past the end repeat the last whole-or-part piece
  const int64_t wstep = 64 * wld * 2, xstep = DW ? 64 * xld * 2 : kStep;  // bytes a step
  uint32_t woff[L], xoff[L];
#pragma unroll
  for (int q = 0; q < L; ++q) {
    const int p = q * BT + tid, r = p >> 5, c = ((((p >> 1) & 15) ^ turn_of(r)) << 4) + (p & 1) * 8;
    woff[q] = (uint32_t)(r * wld + (DMA ? min(c, (cols - 1) & ~7) : min(c, cols))) * 2;
    const int xrow = p >> 3;
    xoff[q] = DW ? (uint32_t)(r * xld + (DMA ? min(c, (rows - 1) & ~7) : min(c, rows))) * 2
                 : (uint32_t)(min(xrow, rows - 1) * xld) * 2 + (((p & 7) ^ (xrow & 7)) << 4);
  }
  // copies q and q + L of a step; the bases move with the steps (a group's rows may span more than 4 GB)
  const uint32_t wat = turned_at<T>(wn, lane), xat = turned_at<T>(wm, lane);
  const uint8_t *xp = (const uint8_t*)xsrc0, *wp = (const uint8_t*)wsrc0;
  // piece q of a turned operand, whose row has `n` columns (without DMA: any alignment, nothing read behind them)
  auto turned_piece = [&](const uint8_t* p, uint32_t off, int q, int n) {
    const int slot = q * BT + tid, c = ((((slot >> 1) & 15) ^ turn_of(slot >> 5)) << 4) + (slot & 1) * 8;
    return load16(p + off, 2 * (n - c), 2 * n);
  };
  auto copy = [&](int q, __amdgpu_buffer_rsrc_t xr, __amdgpu_buffer_rsrc_t wr, uint8_t* d, uint4* hold)
      __attribute__((always_inline)) {
    if constexpr (DMA) {
      to_lds(xr, d + (q * BT + wave * 64) * 16, xoff[q], 0);
      to_lds(wr, d + XB + (q * BT + wave * 64) * 16, woff[q], 0);
    } else {
      if constexpr (DW) hold[q] = turned_piece(xp, xoff[q], q, rows);
      else __builtin_memcpy(hold + q, xp + xoff[q], 16);
      hold[L + q] = turned_piece(wp, woff[q], q, cols);
    }
  };
  auto keep = [&](uint8_t* d, const uint4* hold) __attribute__((always_inline)) {
    if constexpr (!DMA) {
#pragma unroll
      for (int q = 0; q < 2 * L; ++q) *(uint4*)(d + (q * BT + tid) * 16) = hold[q];
    }
  };
  f4v acc[IT][JT];
#pragma unroll
  for (int i = 0; i < IT; ++i)
#pragma unroll
    for (int j = 0; j < JT; ++j) acc[i][j] = f4v{0, 0, 0, 0};
  auto step = [&](auto more, const uint8_t* __restrict st, uint8_t* __restrict nx) __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t xr = rows_at(xp, 0xffffffff), wr = rows_at(wp, 0xffffffff);
    uint32_t at = wat, bt = xat;
    asm volatile("" : "+v"(at), "+v"(bt));  // the addresses are made in the step, not kept across it
    Frag<IN> b[JT], a[2];
    uint4 hold[2 * L];
#pragma unroll
    for (int j = 0; j < JT; ++j) {
      if constexpr (DW) b[j] = frag_turned<IN, T>(st, bt ^ (j << 5));
      else b[j] = frag<IN>(st, wm + j * 16 + lr, lg);
    }
    a[0] = frag_turned<IN, T>(st + XB, at);
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      if (i + 1 < IT) a[(i + 1) & 1] = frag_turned<IN, T>(st + XB, at ^ ((i + 1) << 5));
#pragma unroll
      for (int j = 0; j < JT; ++j) acc[i][j] = mma<IN>(a[i & 1], b[j], acc[i][j]);
      if constexpr (decltype(more)::value) {
        if (i < L) copy(i, xr, wr, nx, hold);
      }
      __builtin_amdgcn_sched_barrier(0);  // rows of tiles stay in this order
    }
    if constexpr (decltype(more)::value) keep(nx, hold);
  };
  static_assert(L <= IT, "two copies with each row of tiles");
  if (steps > 0) {
    const __amdgpu_buffer_rsrc_t xr = rows_at(xp, 0xffffffff), wr = rows_at(wp, 0xffffffff);
    uint4 hold[2 * L];
#pragma unroll
    for (int q = 0; q < L; ++q) copy(q, xr, wr, smem, hold);
    keep(smem, hold);
  }
  const int64_t left = steps_of - (int64_t)steps * 64;
  for (int kt = 0; kt < steps - 1; ++kt) {
    // step kt has landed, and every wave is done with step kt - 1, whose slot the next copies overwrite
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    xp += xstep;
    wp += wstep;
    step(std::true_type(), smem + (kt & 1) * STAGE, smem + (~kt & 1) * STAGE);
  }
  for (int kt = max(0, steps - 1); kt < steps + (left > 0); ++kt) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    uint8_t* d = smem + (kt & 1) * STAGE;
    if (kt == steps) {  // the last, partial step: rows (or columns) of the contraction past the end are zeros
#pragma unroll
      for (int q = 0; q < L; ++q) {
        const int p = q * BT + tid;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        *(uint4*)(d + XB + p * 16) = (p >> 5) >= left ? zero : DMA ? *(const uint4*)(wp + woff[q]) : turned_piece(wp, woff[q], q, cols);
        if constexpr (DW) {
          *(uint4*)(d + p * 16) = (p >> 5) >= left ? zero : DMA ? *(const uint4*)(xp + xoff[q]) : turned_piece(xp, xoff[q], q, rows);
        } else {
          const int c = (p & 7) ^ ((p >> 3) & 7);
          *(uint4*)(d + p * 16) = load16(xp + xoff[q], 2 * (left - c * 8), 2 * steps_of);
        }
      }
      __syncthreads();
    }
    step(std::false_type(), d, smem);
    xp += xstep;
    wp += wstep;
  }
  __syncthreads();  // every wave is done with the last stage
  store_tiles(acc, out, dt, out0 + row0 * ldo + c0, ldo, rows, cols, wn, wm, lr, lg, nullptr, smem + wave * kRowsLds);
}

// dw[g][n][k] = sum over the parts, in order
template <int DT>
__global__ __launch_bounds__(256) void dw_join_kernel(const float* part, int64_t parts, int64_t G, int64_t N, int64_t K,
                                                      void* dw, int64_t ldo, int64_t og) {
  const int64_t each = G * N * K;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < each; i += (int64_t)gridDim.x * 256) {
    float a = 0.0f;
#pragma unroll 4
    for (int64_t p = 0; p < parts; ++p) a += part[p * each + i];
    const int64_t r = i / K, g = r / N;
    put<DT>(dw, g * og + (r - g * N) * ldo + (i - r * K), a);
  }
}

// Both gradients in one grid (dw's tiles first): the workgroups that find no more tiles of the one
// take those of the other, where two launches leave part of the CUs idle at the end of each.
template <int IN, bool DMA>
__global__ __launch_bounds__(512, 2) void grad_kernel(GradArgs A, int dt, int64_t ctiles, int64_t rtiles, int64_t dw_tiles) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  __shared__ int sums[8];
  __shared__ Runs runs[512];
  __shared__ Tile found;
  if (blockIdx.x < dw_tiles) grad_tile<IN, true, DMA>(A, dt, blockIdx.x, ctiles, rtiles, smem, sums, runs, &found);
  else grad_tile<IN, false, DMA>(A, dt, blockIdx.x - dw_tiles, ctiles, 0, smem, sums, runs, &found);
}

int check_out(const char* what, int dt) {
  TRK_REQUIRE(dt == TRK_F32 || dt == TRK_BF16 || dt == TRK_F16, "%s: output must be TRK_F32, TRK_BF16 or TRK_F16", what);
  return TRK_OK;
}

int check_mm(const char* what, const MmArgs& A, int64_t item, bool scaled) {
  TRK_REQUIRE(A.M >= 0 && A.N >= 0 && A.K >= 0 && A.M < ((int64_t)1 << 31) && A.N < ((int64_t)1 << 31) &&
                  A.K < ((int64_t)1 << 31),
              "%s: bad shape M=%lld N=%lld K=%lld", what, (long long)A.M, (long long)A.N, (long long)A.K);
  if (A.M == 0 || A.N == 0) return TRK_OK;
  TRK_REQUIRE(A.y && (A.K == 0 || (A.x && A.w)) && (!scaled || A.K == 0 || (A.sx && A.sw)), "%s: null pointer", what);
  TRK_REQUIRE(A.ldx >= A.K * item && A.ldw >= A.K * item && A.ldy >= A.N, "%s: row stride below the row's length", what);
  // offsets inside a tile of 256 rows are 32 bits
  if (A.ldx >= (1 << 24) || A.ldw >= (1 << 24)) {
    set_error("%s: row strides of 16 MiB and more are not supported", what);
    return TRK_EUNSUPPORTED;
  }
  return TRK_OK;
}

// the steps of a part of rows of `kbytes`, and as many parts as have any
int check_parts(const char* what, int64_t kbytes, const float* part, int64_t& parts, int& share) {
  const int64_t steps = (kbytes + kStep - 1) / kStep;
  TRK_REQUIRE(parts == 1 || (parts > 1 && part && parts <= steps && parts <= 4096),
              "%s: parts must be 1, or at most the blocks of K with the workspace part", what);
  share = parts > 1 ? (int)((steps + parts - 1) / parts) : 0;
  if (parts > 1) parts = (steps + share - 1) / share;
  return TRK_OK;
}

// whole 16-byte pieces of every row at multiples of 16 bytes (offsets inside a tile are 32 bits)
bool rows_aligned(const void* p, int64_t ld) { return aligned16_ptr(p) && ld % 8 == 0; }
bool grad_aligned(const GradArgs& A) {
  return rows_aligned(A.dy, A.ldy) && (!A.dw || rows_aligned(A.x, A.ldx)) &&
         (!A.dx || (rows_aligned(A.w, A.ldw) && A.wg % 8 == 0));
}

// Facts of the current device, asked for once each: its CUs, and that a kernel F may have more than 64 KB of
// shared memory.
struct Device {
  int id = 0, cus = 256;
};
Device current_device() {
  static std::atomic<int> known[64];
  Device d;
  if (hipGetDevice(&d.id) != hipSuccess) d.id = 0;
  int n = d.id < 64 ? known[d.id].load(std::memory_order_relaxed) : 0;
  if (n == 0 && hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, d.id) == hipSuccess && d.id < 64)
    known[d.id].store(n, std::memory_order_relaxed);
  if (n > 0) d.cus = n;
  return d;
}
template <typename F>
bool allow_lds(F* f, int bytes, const Device& d, std::atomic<uint64_t>& allowed) {
  const uint64_t bit = d.id < 64 ? 1ull << d.id : 0;
  if (bit & allowed.load(std::memory_order_relaxed)) return true;
  if (hipFuncSetAttribute((const void*)f, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) return false;
  allowed.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

// row tiles there can be: at most M groups have rows, each with at most one part tile, and the rows behind them
// have one
int64_t row_tiles(const MmArgs& A, int tm) {
  return A.counts ? A.M / tm + std::min(A.G, A.M) + 1 : (A.M + tm - 1) / tm;
}

template <int IN>
int launch_grad(const char* what, const GradArgs& A, int dt, hipStream_t st) {
  constexpr int T = 256, lds = 4 * T * kStep;
  static std::atomic<uint64_t> allowed[2];
  const bool al = grad_aligned(A);
  auto* f = al ? grad_kernel<IN, true> : grad_kernel<IN, false>;
  TRK_REQUIRE(allow_lds(f, lds, current_device(), allowed[al]), "%s: %d bytes of shared memory are not available", what, lds);
  const int64_t ct = (A.K + T - 1) / T, rt = (A.N + T - 1) / T;
  // (whole rounds over the XCDs, so that both lists of tiles start at the first one)
  const int64_t dw = A.dw ? (ct * rt * A.G * A.parts + 7) / 8 * 8 : 0, dx = A.dx ? ct * (A.M / T + std::min(A.G, A.M) + 1) : 0;
  TRK_REQUIRE(dw + dx < (1 << 23), "%s: too many tiles", what);  // (2^32 threads)
  f<<<(unsigned)(dw + dx), 512, lds, st>>>(A, dt, ct, rt, dw);
  if (A.dw && A.parts > 1) {
    const unsigned blocks = (unsigned)std::min<int64_t>((A.G * A.N * A.K + 255) / 256, 4096);
    dw_join_kernel<IN == IN_BF16 ? TRK_BF16 : TRK_F16><<<blocks, 256, 0, st>>>(A.part, A.parts, A.G, A.N, A.K, A.dw, A.ldo, A.og);
  }
  return trk::check_launch(what);
}

// row tiles that have rows, as far as the host knows: groups have at least a tile each
int64_t live_tiles(int64_t G, int64_t M, int tm) { return std::max((M + tm - 1) / tm, std::min(G, M)); }

// Few strips of 16 JT rows x 16 columns: straight from memory to registers, 16 rows a strip while there
// are at most 256, else the fewest strips by the work of one (1, 1.4 and 2.2 for 16, 32 and 64 rows).
// In 8 bits, us, strips / 128-tiles: 16 x 4096 x 4096 7.0 / 20.9, 64 x 4096 x 4096 13.9 / 21.0, 256 x
// 1024 x 1024 6.2 / 8.6, 32 x 16384 x 4096 26.5 / 28.5; past the limits 128 x 4096 x 4096 22.8 / 21.2,
// 16 x 50000 x 1024 18.0 / 12.7, 512 x 8192 x 1024 40.7 / 10.5.  JT, or 0: tiles.
int few_strips(int64_t G, int64_t M, int64_t N) {
  const int64_t strips = (N + 15) / 16, s16 = strips * live_tiles(G, M, 16), s32 = strips * live_tiles(G, M, 32),
                s64 = strips * live_tiles(G, M, 64);
  if (s16 <= 256 || (s16 <= 1024 && 5 * s16 <= 7 * s32 && 5 * s16 <= 11 * s64)) return 1;
  if (s32 <= 1024 && 7 * s32 <= 11 * s64) return 2;
  return s64 <= 512 ? 4 : 0;
}

// Few 128-tiles (of even groups) and long rows: K in parts, as many as give 384 tiles of at least 8 steps, up to 8.
// In 16 / 8 bits, us, 1 part / the rule's: 8 groups, 512 x 2048 x 8192 115 / 66 and 55 / 36; 1000 x 1024 x 8192 in 4
// 83 / 38 and 54 / 29; 600 x 1024 x 16384 in 2 162 / 50 and 100 / 36; 600 x 928 x 6288 90 / 32 and 57 / 25; 1000 x
// 1000 x 2048 28 / 22 in 16 bits, in 8 (16 steps) 18 against 22 in 4 parts; 16 x 20000 x 8192 128 / 85 and 52 / 38, 8
// groups, 16 x 2304 x 8192 122 / 78 and 54 / 40.  Rows that strips of 16 take stay whole
// (8 groups, 64 x 2048 x 8192 52 against 56 in 3 parts), and up to 64 steps 256 strips of 64 (64 x 4096 x 4096 24 /
// 19 in 16 bits, 17 / 18 in 8).  The join takes 4 to 6 us of it, and a launch.
int64_t parts_of(int64_t G, int64_t M, int64_t N, int64_t steps) {
  if (G < 1 || M < 1 || N < 1 || steps <= 24) return 1;
  const int64_t groups = std::min(G, M), tiles = groups * (((M + groups - 1) / groups + 127) / 128) * ((N + 127) / 128);
  if (tiles > 192 || few_strips(G, M, N) == 1) return 1;
  if (steps <= 64 && (N + 15) / 16 * live_tiles(G, M, 64) <= 256) return 1;
  return std::min({384 / tiles, steps / 8, (int64_t)8});
}

template <int IN, bool WROW, int JT>
int launch_few(const char* what, const MmArgs& A, int dt, hipStream_t st) {
  const int64_t strips = (A.N + 15) / 16, live = live_tiles(A.G, A.M, 16 * JT), steps = (A.K * (is8(IN) ? 1 : 2) + kStep - 1) / kStep;
  // Waves that share 16 columns: enough for 2048 waves in all, and no more than there are steps (one step: 1).  Few
  // strips come here (1024 at most), so the first rule ends at 2.  16 rows, us with 2 / 4 / 8: 4096 x 4096 in 8 bits
  // 17.8 / 10.8 / 7.0, in 16 32.4 / 18.9 / 12.2; 8192 x 4096 18.8 / 11.2 / 10.9, 32.6 / 19.5 / 21.7; 16384 x 4096
  // 19.4 / 18.4 / 19.0, 32.9 / 35.8 / 39.1
  int kw = 8;
  while (kw > 1 && (strips * live * (kw / 2) >= 2048 || kw > steps)) kw /= 2;
  const dim3 grid((unsigned)((strips + 8 / kw - 1) / (8 / kw)), (unsigned)row_tiles(A, 16 * JT));
  if (kw == 8) mm_few_kernel<IN, WROW, JT, 8><<<grid, 512, 0, st>>>(A, dt);
  else if (kw == 4) mm_few_kernel<IN, WROW, JT, 4><<<grid, 512, 0, st>>>(A, dt);
  else if (kw == 2) mm_few_kernel<IN, WROW, JT, 2><<<grid, 512, 0, st>>>(A, dt);
  else mm_few_kernel<IN, WROW, JT, 1><<<grid, 512, 0, st>>>(A, dt);
  return trk::check_launch(what);
}

template <int IN, bool WROW, bool DMA, int T, int WN, int WM>
int launch_tile(const char* what, const MmArgs& A, int dt, const Device& dev, hipStream_t st) {
  static std::atomic<uint64_t> allowed{0};
  constexpr int BT = WN * WM * 64;
  constexpr int lds = 2 * (2 * T * kStep + (is8(IN) ? (2 * T + BT - 1) / BT * BT * 4 : 0));
  auto* f = mm_tile_kernel<IN, WROW, DMA, T, T, WN, WM>;
  TRK_REQUIRE(allow_lds(f, lds, dev, allowed), "%s: %d bytes of shared memory are not available", what, lds);
  const int64_t nt = (A.N + T - 1) / T, mt = row_tiles(A, T);
  TRK_REQUIRE(nt * mt * A.parts < ((int64_t)1 << 31), "%s: too many tiles", what);
  const int64_t grid = std::min<int64_t>(nt * mt * A.parts, (int64_t)dev.cus * (BT == 256 ? 2 : 1) / 8 * 8);
  f<<<(unsigned)grid, BT, lds, st>>>(A, dt, (int)nt, (int)mt);
  return trk::check_launch(what);
}

template <int IN, bool WROW>
int launch_tiles(const char* what, const MmArgs& A, int dt, bool aligned, float* part, hipStream_t st) {
  const Device dev = current_device();
  if (A.parts > 1) {
    MmArgs P = A;
    P.y = part;
    P.ldy = A.N;
    P.bias = nullptr;
    P.zero_tail = 0;
    if (int rc = aligned ? launch_tile<IN, WROW, true, 128, 2, 2>(what, P, TRK_F32, dev, st)
                         : launch_tile<IN, WROW, false, 128, 2, 2>(what, P, TRK_F32, dev, st))
      return rc;
    const unsigned blocks = (unsigned)std::min<int64_t>((A.M * ((A.N + 3) / 4) + 255) / 256, 8 * dev.cus);
    mm_join_kernel<<<blocks, 256, 0, st>>>(A, part, dt);
    return trk::check_launch(what);
  }
  switch (few_strips(A.G, A.M, A.N)) {  // (the grid's second length is below 4096)
    case 1: return launch_few<IN, WROW, 1>(what, A, dt, st);
    case 2: return launch_few<IN, WROW, 2>(what, A, dt, st);
    case 4: return launch_few<IN, WROW, 4>(what, A, dt, st);
  }
  // 256-tiles where whole ones alone fill the CUs, of even groups (a tile has rows of one): 2048 x 8192 x 1024 in 8 bits
  // 23.2 us against 25.8 with 128-tiles, 1024 x 8192 x 1024 20.2 against 15.2.  64 groups x 2048 x 1024 in 8 / 16
  // bits, 256 against 128: of 128 rows each 46 / 80 against 39 / 67, of 256 50 / 92 against 55 / 104, of 1024 189 / 303
  // against 251 / 352; 256 groups of 32 rows 168 / 291 against 136 / 218.  What counts is not known here where
  // groups are ragged: 256 rows on average 78 / 133 against 68 / 120, 1024 222 / 333 against 263 / 370.  f32
  // outputs have wider fragments, and unaligned 8-bit rows are held in registers on their way: both leave
  // room for 128-tiles only.
  if constexpr (IN != IN_E4M3X) {
    const int64_t groups = std::min(A.G, A.M);
    if ((A.N + 255) / 256 * (groups * (A.M / groups / 256)) >= dev.cus) {
      if (aligned) return launch_tile<IN, WROW, true, 256, 2, 4>(what, A, dt, dev, st);
      if constexpr (!is8(IN)) return launch_tile<IN, WROW, false, 256, 2, 4>(what, A, dt, dev, st);
    }
  }
  return aligned ? launch_tile<IN, WROW, true, 128, 2, 2>(what, A, dt, dev, st)
                 : launch_tile<IN, WROW, false, 128, 2, 2>(what, A, dt, dev, st);
}

int launch_mm(const char* what, const MmArgs& A, int in, int wrow, int dt, float* part, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  const bool al = aligned16_ptr(A.x) && aligned16_ptr(A.w) && A.ldx % 16 == 0 && A.ldw % 16 == 0 && A.wg % 16 == 0;
  if (in == IN_E4M3 && dt == TRK_F32)
    return wrow ? launch_tiles<IN_E4M3X, true>(what, A, dt, al, part, st) : launch_tiles<IN_E4M3X, false>(what, A, dt, al, part, st);
  if (in == IN_E4M3)
    return wrow ? launch_tiles<IN_E4M3, true>(what, A, dt, al, part, st) : launch_tiles<IN_E4M3, false>(what, A, dt, al, part, st);
  if (in == IN_BF16) return launch_tiles<IN_BF16, false>(what, A, dt, al, part, st);
  return launch_tiles<IN_F16, false>(what, A, dt, al, part, st);
}

}  // namespace

extern "C" {

int64_t trk_matmul_fp8_parts(int64_t M, int64_t N, int64_t K) { return parts_of(1, M, N, (K + kStep - 1) / kStep); }

int trk_matmul_fp8(const void* x, int64_t ldx, const float* sx, int64_t sx_row, int64_t sx_kb, const void* w,
                   int64_t ldw, const float* sw, int64_t sw_row, int64_t sw_kb, int w_block_rows, const float* bias,
                   int64_t M, int64_t N, int64_t K, void* y, int64_t ldy, int out_dtype, float* part, int64_t parts,
                   void* stream) {
  const char* what = "trk_matmul_fp8";
  if (int rc = check_out(what, out_dtype)) return rc;
  TRK_REQUIRE(w_block_rows == 1 || w_block_rows == 128, "%s: w_block_rows must be 1 or 128", what);
  int share;
  if (int rc = check_parts(what, K, part, parts, share)) return rc;
  const MmArgs A{(const uint8_t*)x, (const uint8_t*)w, sx, sw, bias, y, nullptr, ldx, ldw, 0, sx_row, sx_kb,
                 sw_row, sw_kb, 0, ldy, M, N, K, 1, 0, (int)parts, share};
  if (int rc = check_mm(what, A, 1, true)) return rc;
  if (M == 0 || N == 0) return TRK_OK;
  return launch_mm(what, A, IN_E4M3, w_block_rows == 1, out_dtype, part, stream);
}

int64_t trk_matmul_grouped_parts(int64_t G, int64_t M, int64_t N, int64_t K, int in_dtype) {
  return parts_of(G, M, N, (K * (in_dtype == TRK_E4M3 ? 1 : 2) + kStep - 1) / kStep);
}

int trk_matmul_grouped_split(const void* x, int64_t ldx, const float* sx, int64_t sx_row, int64_t sx_kb, const void* w,
                             int64_t ldw, int64_t wg, const float* sw, int64_t sw_row, int64_t sw_kb, int64_t sw_g,
                             int w_block_rows, const int32_t* counts, int64_t G, int64_t M, int64_t N, int64_t K,
                             int in_dtype, void* y, int64_t ldy, int out_dtype, int zero_tail, float* part, int64_t parts,
                             void* stream) {
  const char* what = "trk_matmul_grouped";
  if (int rc = check_out(what, out_dtype)) return rc;
  TRK_REQUIRE(in_dtype == TRK_E4M3 || in_dtype == TRK_BF16 || in_dtype == TRK_F16,
              "%s: input must be TRK_E4M3, TRK_BF16 or TRK_F16", what);
  const bool f8 = in_dtype == TRK_E4M3;
  TRK_REQUIRE(!f8 || w_block_rows == 1 || w_block_rows == 128, "%s: w_block_rows must be 1 or 128", what);
  TRK_REQUIRE(G >= 1 && G <= 65535 && counts, "%s: 1 to 65535 groups and their counts are required", what);
  const int64_t item = f8 ? 1 : 2;
  int share;
  if (int rc = check_parts(what, K * item, part, parts, share)) return rc;
  const MmArgs A{(const uint8_t*)x, (const uint8_t*)w, sx, sw, nullptr, y, counts, ldx * item, ldw * item, wg * item,
                 sx_row, sx_kb, sw_row, sw_kb, sw_g, ldy, M, N, K, G, zero_tail, (int)parts, share};
  if (int rc = check_mm(what, A, item, f8)) return rc;
  if (M == 0 || N == 0) return TRK_OK;
  return launch_mm(what, A, f8 ? IN_E4M3 : in_dtype == TRK_BF16 ? IN_BF16 : IN_F16, f8 && w_block_rows == 1, out_dtype,
                   part, stream);
}

int trk_matmul_grouped(const void* x, int64_t ldx, const float* sx, int64_t sx_row, int64_t sx_kb, const void* w,
                       int64_t ldw, int64_t wg, const float* sw, int64_t sw_row, int64_t sw_kb, int64_t sw_g,
                       int w_block_rows, const int32_t* counts, int64_t G, int64_t M, int64_t N, int64_t K, int in_dtype,
                       void* y, int64_t ldy, int out_dtype, int zero_tail, void* stream) {
  return trk_matmul_grouped_split(x, ldx, sx, sx_row, sx_kb, w, ldw, wg, sw, sw_row, sw_kb, sw_g, w_block_rows, counts, G, M,
                                  N, K, in_dtype, y, ldy, out_dtype, zero_tail, nullptr, 1, stream);
}

// Few tiles and many rows: a group's rows are split into parts, so that the tiles fill the CUs, of at least 4 steps
// of 64 rows on average (3 groups of 9082 rows in all, 121 x 102, with forward and autograd: 619 us in one
// part, under 110 in 11).
int64_t trk_matmul_grouped_bwd_parts(int64_t G, int64_t M, int64_t N, int64_t K) {
  if (G < 1 || M < 1 || N < 1 || K < 1) return 1;
  const int64_t tiles = (N + 255) / 256 * ((K + 255) / 256) * G;
  return std::max<int64_t>(1, std::min(256 / tiles, M / (G * 256)));
}

int trk_matmul_grouped_bwd(const void* dy, int64_t ldy, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t wg,
                           const int32_t* counts, int64_t G, int64_t M, int64_t N, int64_t K, int dtype, void* dx,
                           int64_t lddx, void* dw, int64_t lddw, int64_t dwg, float* part, int64_t parts, void* stream) {
  const char* what = "trk_matmul_grouped_bwd";
  TRK_REQUIRE(dtype == TRK_BF16 || dtype == TRK_F16, "%s: dtype must be TRK_BF16 or TRK_F16", what);
  TRK_REQUIRE(G >= 1 && G <= 65535 && counts, "%s: 1 to 65535 groups and their counts are required", what);
  TRK_REQUIRE(M >= 0 && N >= 0 && K >= 0 && M < ((int64_t)1 << 31) && N < ((int64_t)1 << 31) && K < ((int64_t)1 << 31),
              "%s: bad shape M=%lld N=%lld K=%lld", what, (long long)M, (long long)N, (long long)K);
  if (M == 0 || K == 0) dx = nullptr;
  if (N == 0 || K == 0) dw = nullptr;
  if (!dx && !dw) return TRK_OK;
  TRK_REQUIRE(M == 0 || N == 0 || dy, "%s: null pointer", what);
  TRK_REQUIRE(M == 0 || N == 0 || ((!dx || w) && (!dw || x)), "%s: null pointer", what);
  TRK_REQUIRE(ldy >= N && (!dx || (ldw >= K && lddx >= K)) && (!dw || (ldx >= K && lddw >= K)),
              "%s: row stride below the row's length", what);
  if (ldy >= (1 << 23) || (dx && ldw >= (1 << 23)) || (dw && ldx >= (1 << 23))) {
    set_error("%s: row strides of 16 MiB and more are not supported", what);
    return TRK_EUNSUPPORTED;
  }
  TRK_REQUIRE(parts >= 1 && parts <= 4096 && (parts == 1 || !dw || part), "%s: parts > 1 need the workspace part", what);
  const GradArgs A{(const uint16_t*)dy, (const uint16_t*)x, (const uint16_t*)w, dx, dw, counts, ldy, ldx, ldw, wg, lddx,
                   lddw, dwg, M, N, K, G, part, parts};
  hipStream_t st = (hipStream_t)stream;
  return dtype == TRK_BF16 ? launch_grad<IN_BF16>(what, A, dtype, st) : launch_grad<IN_F16>(what, A, dtype, st);
}

}  // extern "C"
