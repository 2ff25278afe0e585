// Shared parts of the ragged cross-attention kernels (cross_attn_fwd.hip, cross_attn_bwd.hip).
//
//   z_ij = scale q_i . k_j + table[h, bucket(i, j)],  p = softmax_j z,  o_i = sum_j p_ij v_j
//
// over the keys j of row i's own sequence.  Every product runs on the matrix units with the score
// tile TRANSPOSED onto the next product's operand: a 16x16 result tile has its column in
// lane & 15 and its rows 4 (lane >> 4) + r in four registers, and a right-hand operand has its
// column in lane & 15 and its contraction index in registers.  So S^T = K Q^T (or S = Q K^T in the
// key-owned pass) feeds V^T P^T (or dO^T P) straight from registers: the scores never visit LDS,
// and a query row's running maximum is one value a lane.  The contraction index of that second
// product is permuted (4 g + r of two 16-row blocks), which costs nothing because the left-hand
// operand is read from LDS with the same permutation.
//
//   float:      v_mfma_f32_16x16x4 (exact fp32 products; fp32 rate)
//   bf16, fp16: v_mfma_f32_16x16x32 with fp32 accumulators; the left-hand operand of the second
//               product is read transposed by ds_read_b64_tr_b16
#pragma once

#include "ragged.h"

namespace hy {
namespace xa {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef short s8v __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s4v lds_s4v;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMaxBuckets = 64;  // the gradient keeps one column a lane of a [buckets, 64] table in LDS
constexpr int kMaxFar = 2048;    // the bias is looked up by whole distance in LDS
constexpr int kTile = 64;        // rows of the operand that is streamed through LDS

enum Bias { kNoBias = 0, kOrder = 1, kSpace = 2 };

// The bucket of a whole distance n: n itself below `near`, then one more for each threshold reached.
struct Rule {
  int buckets;    // columns of the table
  int side;       // buckets of one direction (order, two sided), else all of them
  int near, far;  // distances from `far` on share the last bucket
  int two_sided;
  int nthr;
  int thr[kMaxBuckets];
  float inv_unit;
  double unit;
};

struct Args {
  const void *q, *k, *v;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // strides in elements
  const int *q_ptr, *k_ptr;
  const uint8_t* key_mask;
  int Nq, Nk, S, H, Hk, G, D;
  int vec_q, vec_k, vec_v, vec_do;  // rows may be read 16 bytes at a time
  float scale;
  void* out;    // [Nq, H, D]
  void* rest;   // [Nq, H, D], 16-bit types in training: what the rounding of `out` leaves.  The backward's
                // delta = do . o is exact with it: dS = p (dP - delta) cancels where a row's dP are near
                // each other, and the bias' gradient sums such dS over whole buckets.
  float* lse;   // [H, Nq], log2 of the row's sum; +inf where no key is
  const void* table;  // [H, buckets] fp32
  const void *q_pos, *k_pos;
  Rule rule;
  // backward
  const void* d_out;
  int64_t do_row, do_head;
  float* delta;  // [H, Nq]
  void *dq, *dk, *dv;  // [Nq, H, D], [Nk, Hk, D] x 2
  float* part;   // [tiles, H, buckets]
};

// ------------------------------------------------------------------ operands
template <typename T>
struct El;
template <>
struct El<float> {
  static constexpr int kPer = 4;  // elements of 16 bytes
};
template <>
struct El<__bf16> {
  static constexpr int kPer = 8;
  typedef b8 v8;
  typedef b4 v4;
  static __device__ __forceinline__ f4 mfma(b8 a, b8 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct El<_Float16> {
  static constexpr int kPer = 8;
  typedef h8 v8;
  typedef h4 v4;
  static __device__ __forceinline__ f4 mfma(h8 a, h8 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

// 16 bytes of row `p` from column d0 on; zeros behind column D (and where !ok)
template <typename T>
__device__ __forceinline__ uint4 load16(const T* p, int d0, int D, bool ok, bool vec) {
  uint4 r = make_uint4(0, 0, 0, 0);
  if (!ok || d0 >= D) return r;
  if (vec) return *reinterpret_cast<const uint4*>(p + d0);
  constexpr int kPer = El<T>::kPer;
  union {
    uint4 u;
    T e[kPer];
  } x;
  x.u = r;
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (d0 + i < D) x.e[i] = p[d0 + i];
  return x.u;
}

// One operand of width DP (the head width rounded up) in LDS or registers.
//   Row:   the operand of a product that contracts over the width; lane & 15 is its row, and
//          the width goes over lane >> 4 and registers in the same order on both sides.
//   outer: products that contract over 32 rows of an LDS tile, into [width, 16] accumulators.
template <typename T, int DP>
struct Mat {
  typedef typename El<T>::v8 v8;
  static constexpr int LD = DP + 8;  // a stride of 4 banks beyond a multiple of 64: 16 rows meet no bank twice
  static constexpr int RF = DP / 32, DT = DP / 16;
  struct Row {
    v8 f[RF];
  };
  static __device__ __forceinline__ Row row_lds(const T* row, int g) {
    Row x;
#pragma unroll
    for (int j = 0; j < RF; ++j) x.f[j] = *reinterpret_cast<const v8*>(row + 32 * j + 8 * g);
    return x;
  }
  static __device__ __forceinline__ Row row_global(const T* row, int g, int D, bool ok, bool vec) {
    Row x;
#pragma unroll
    for (int j = 0; j < RF; ++j) {
      const uint4 u = load16(row, 32 * j + 8 * g, D, ok, vec);
      x.f[j] = __builtin_bit_cast(v8, u);
    }
    return x;
  }
  static __device__ __forceinline__ f4 dot(const Row& a, const Row& b, f4 acc) {
#pragma unroll
    for (int j = 0; j < RF; ++j) acc = El<T>::mfma(a.f[j], b.f[j], acc);
    return acc;
  }
  // acc[n][dt] += tile[32 rows]^T p[n]; the products' p is rounded to the operands' type here, and
  // nowhere else (sums and statistics use it unrounded).  FINE: p in two parts, the second what the
  // first leaves, so that its rounding is of the accumulators' order.
  template <int N, bool FINE>
  static __device__ __forceinline__ void outer(const T* tile, const f4 (&p0)[N], const f4 (&p1)[N],
                                               f4 (&acc)[N][DT], int lane) {
    const int g = lane >> 4, li = lane & 15;
    v8 pb[N], pl[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const f8 w = f8{p0[n][0], p0[n][1], p0[n][2], p0[n][3], p1[n][0], p1[n][1], p1[n][2], p1[n][3]};
      pb[n] = __builtin_convertvector(w, v8);
      if constexpr (FINE) pl[n] = __builtin_convertvector(w - __builtin_convertvector(pb[n], f8), v8);
    }
    const T* at = tile + (4 * g + (li >> 2)) * LD + 4 * (li & 3);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const s4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4v*)(at + 16 * dt));
      const s4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4v*)(at + 16 * LD + 16 * dt));
      const v8 a = __builtin_bit_cast(v8, (s8v{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}));
#pragma unroll
      for (int n = 0; n < N; ++n) {
        acc[n][dt] = El<T>::mfma(a, pb[n], acc[n][dt]);
        if constexpr (FINE) acc[n][dt] = El<T>::mfma(a, pl[n], acc[n][dt]);
      }
    }
  }
  // rounds to T; `rest`, if there is one, takes what the rounding leaves
  static __device__ __forceinline__ void store(T* row, const f4 (&acc)[DT], float mul, int D, int g,
                                               T* rest = nullptr) {
    typedef typename El<T>::v4 v4;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const int d = 16 * dt + 4 * g;
      const f4 x = acc[dt] * mul;
      const v4 y = __builtin_convertvector(x, v4);
      const v4 z = __builtin_convertvector(x - __builtin_convertvector(y, f4), v4);
      if ((D & 3) == 0) {
        if (d < D) {
          *reinterpret_cast<v4*>(row + d) = y;
          if (rest != nullptr) *reinterpret_cast<v4*>(rest + d) = z;
        }
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (d + r < D) {
            row[d + r] = y[r];
            if (rest != nullptr) rest[d + r] = z[r];
          }
      }
    }
  }
};

template <int DP>
struct Mat<float, DP> {
  static constexpr int LD = DP + 4;
  static constexpr int RF = DP / 16, DT = DP / 16;
  static constexpr int VW = DT < 4 ? DT : 4, JJ = DT / VW;  // columns of one read, and reads, of `outer`
  struct Row {
    f4 f[RF];
  };
  static __device__ __forceinline__ Row row_lds(const float* row, int g) {
    Row x;
#pragma unroll
    for (int j = 0; j < RF; ++j) x.f[j] = *reinterpret_cast<const f4*>(row + 16 * j + 4 * g);
    return x;
  }
  static __device__ __forceinline__ Row row_global(const float* row, int g, int D, bool ok, bool vec) {
    Row x;
#pragma unroll
    for (int j = 0; j < RF; ++j) x.f[j] = __builtin_bit_cast(f4, load16(row, 16 * j + 4 * g, D, ok, vec));
    return x;
  }
  static __device__ __forceinline__ f4 dot(const Row& a, const Row& b, f4 acc) {
#pragma unroll
    for (int j = 0; j < RF; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.f[j][i], b.f[j][i], acc, 0, 0, 0);
    return acc;
  }
  template <int N, bool FINE>  // one part is exact
  static __device__ __forceinline__ void outer(const float* tile, const f4 (&p0)[N], const f4 (&p1)[N],
                                               f4 (&acc)[N][DT], int lane) {
    const int g = lane >> 4, li = lane & 15;
    typedef float vw __attribute__((ext_vector_type(VW)));
    const float* at = tile + 4 * g * LD + VW * li;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int jj = 0; jj < JJ; ++jj) {
          float a[VW];
          const float* from = at + (16 * t + r) * LD + 64 * jj;
          if constexpr (VW == 1) {
            a[0] = *from;
          } else {
            const vw x = *reinterpret_cast<const vw*>(from);
#pragma unroll
            for (int i = 0; i < VW; ++i) a[i] = x[i];
          }
#pragma unroll
          for (int i = 0; i < VW; ++i)
#pragma unroll
            for (int n = 0; n < N; ++n)
              acc[n][jj * VW + i] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], t ? p1[n][r] : p0[n][r],
                                                                         acc[n][jj * VW + i], 0, 0, 0);
        }
  }
  // accumulator jj * VW + i, register r: column 64 jj + (4 g + r) VW + i
  static __device__ __forceinline__ void store(float* row, const f4 (&acc)[DT], float mul, int D, int g,
                                               float* = nullptr) {
#pragma unroll
    for (int jj = 0; jj < JJ; ++jj)
#pragma unroll
      for (int c = 0; c < VW; ++c) {
        const int d = 64 * jj + 4 * g * VW + 4 * c;
        f4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = acc[jj * VW + (4 * c + e) % VW][(4 * c + e) / VW] * mul;
        if ((D & 3) == 0) {
          if (d < D) *reinterpret_cast<f4*>(row + d) = x;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (d + e < D) row[d + e] = x[e];
        }
      }
  }
};

// One streamed operand's tile of kTile rows on its way from memory to LDS: 256 threads, 16 bytes
// each, held in registers while the tile before it is worked on.  Rows outside [., end) and masked
// ones become zeros, so that whatever they hold (infinities, NaN) meets no product.
template <typename T, int DP>
struct Stage {
  static constexpr int kPer = El<T>::kPer;
  static constexpr int CPR = DP / kPer;                  // 16-byte chunks of a row
  static constexpr int CH = kTile * CPR / 256;           // of one thread
  static_assert(kTile * CPR % 256 == 0, "a tile is a whole number of chunks a thread");
  uint4 r[CH];
  __device__ __forceinline__ void load(const T* base, int64_t stride, int row0, int end, const uint8_t* mask, int D,
                                       bool vec, int tid) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int i = tid + c * 256, row = row0 + i / CPR;
      const bool ok = row < end && (mask == nullptr || mask[row] != 0);
      r[c] = load16(base + (int64_t)row * stride, (i % CPR) * kPer, D, ok, vec);
    }
  }
  __device__ __forceinline__ void store(T* lds, int tid) const {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int i = tid + c * 256;
      *reinterpret_cast<uint4*>(lds + (i / CPR) * Mat<T, DP>::LD + (i % CPR) * kPer) = r[c];
    }
  }
};

// ------------------------------------------------------------------ reductions over a column's four lanes
__device__ __forceinline__ float column_max(float x) {
  const unsigned u = __float_as_uint(x);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const float y = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const unsigned w = __float_as_uint(y);
  const auto b = __builtin_amdgcn_permlane16_swap(w, w, false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

__device__ __forceinline__ float column_sum(float x) {
  const unsigned u = __float_as_uint(x);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const float y = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const unsigned w = __float_as_uint(y);
  const auto b = __builtin_amdgcn_permlane16_swap(w, w, false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// ------------------------------------------------------------------ buckets
__device__ __forceinline__ int bucket_of(const Rule& r, int n) {
  if (n < r.near) return n;
  int b = r.near;
  for (int j = 0; j < r.nthr; ++j) b += n >= r.thr[j] ? 1 : 0;
  return b;
}

template <int BIAS>
__device__ __forceinline__ int lut_size(const Rule& r) {
  return BIAS == kOrder ? 2 * r.far + 1 : r.far + 1;
}

template <int BIAS>
__device__ __forceinline__ int lut_bucket(const Rule& r, int i) {  // bucket of look-up entry i
  if constexpr (BIAS == kOrder) {
    const int rel = i - r.far;
    if (r.two_sided) return bucket_of(r, abs(rel)) + (rel > 0 ? r.side : 0);
    return bucket_of(r, max(-rel, 0));
  } else {
    return bucket_of(r, i);
  }
}

// Entry of a pair by order: whole positions, whose difference may pass 32 bits.
__device__ __forceinline__ int order_index(int kp, int qp, int far) {
  const int rel = __builtin_elementwise_sub_sat(kp, qp);
  return min(max(rel, -far), far) + far;
}

// Entry of a pair by distance: floor(dist / unit).  In fp32 first; where that lies within its own
// rounding (2^-20 relative covers the difference, the squares, the root and 1 / unit) of a whole
// number, again in 64 bits, so that the bucket is the one that 64 bits give, on a lattice too.
__device__ __forceinline__ int space_index(float qx, float qy, float qz, float kx, float ky, float kz, const Rule& r) {
  const float dx = kx - qx, dy = ky - qy, dz = kz - qz;
  const float t = __builtin_amdgcn_sqrtf(fmaf(dx, dx, fmaf(dy, dy, dz * dz))) * r.inv_unit;
  const float far = (float)r.far;
  int i = t < far ? (int)t : r.far;  // not a number: far
  if (fabsf(t - rintf(t)) < t * 0x1p-20f && t < far + 1.f) {
#pragma clang fp contract(off)
    const double ex = (double)kx - (double)qx, ey = (double)ky - (double)qy, ez = (double)kz - (double)qz;
    const double u = __builtin_sqrt(ex * ex + ey * ey + ez * ez) / r.unit;
    i = u < (double)r.far ? (int)u : r.far;
  }
  return i;
}

// Keys' or queries' positions of one streamed tile in LDS (int: one array; space: three).
template <int BIAS>
__device__ __forceinline__ void stage_pos(int* lds, const void* pos, int row0, int end, int tid) {
  if constexpr (BIAS == kOrder) {
    if (tid < kTile) lds[tid] = row0 + tid < end ? ((const int*)pos)[row0 + tid] : 0;
  } else if constexpr (BIAS == kSpace) {
    if (tid < 3 * kTile) {
      const int row = tid / 3, c = tid - 3 * row;
      ((float*)lds)[c * kTile + row] = row0 + row < end ? ((const float*)pos)[(int64_t)(row0 + row) * 3 + c] : 0.f;
    }
  }
}

struct Pos {  // one row's position
  int i;
  float x, y, z;
};

template <int BIAS>
__device__ __forceinline__ Pos load_pos(const void* pos, int row, bool ok) {
  Pos p = {0, 0.f, 0.f, 0.f};
  if (!ok) return p;
  if constexpr (BIAS == kOrder) p.i = ((const int*)pos)[row];
  if constexpr (BIAS == kSpace) {
    const float* f = (const float*)pos + (int64_t)row * 3;
    p.x = f[0];
    p.y = f[1];
    p.z = f[2];
  }
  return p;
}

}  // namespace xa
}  // namespace hy
