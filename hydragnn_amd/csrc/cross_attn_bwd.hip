// Ragged cross attention, backward (see cross_attn.h for the mathematics and the layouts).
//
//   delta_i = do_i . o_i,  p = exp(z - lse),  dS = p (do v^T - delta)
//   dq = scale dS k,  dk = scale dS^T q,  dv = p^T do,  dtable[h, b] = sum of dS over the pairs of bucket b
//
// Two passes, each of which owns what it writes, so that no sum goes by atomics and every run gives
// the same bits: the query pass (dq, delta, the table's sums), whose waves own 16 query rows each and
// stream the keys, and the key pass (dk, dv), whose waves own 16 keys each and stream the queries of
// every head that shares them.
#include "cross_attn.h"

namespace hy {
namespace xa {

// ------------------------------------------------------------------ query pass
template <typename T, int DP, int NQ, int BIAS>
__global__ __launch_bounds__(256) void bwd_query_kernel(Args a) {
  typedef Mat<T, DP> M;
  constexpr int ROWS = 64 * NQ;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  T* Ks = (T*)smem;
  T* Vs = Ks + kTile * M::LD;
  float* kadd = (float*)(Vs + kTile * M::LD);
  int* kpos = (int*)(kadd + kTile);
  float* hist = (float*)(kpos + 3 * kTile);  // [4 waves, buckets, 64 lanes]: every lane adds to its own column
  const int nb = BIAS != kNoBias ? a.rule.buckets : 0;
  float* lut = hist + 4 * nb * 64;
  const int nl = BIAS != kNoBias ? lut_size<BIAS>(a.rule) : 0;
  uint8_t* lutb = (uint8_t*)(lut + nl);

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, li = lane & 15;
  const int h = blockIdx.x % a.H;
  const Tile tile = find_tile(a.q_ptr, a.S, a.Nq, ROWS, blockIdx.x / a.H);
  if (tile.start >= tile.end) {
    if (BIAS != kNoBias && tid < nb) a.part[(int64_t)blockIdx.x * nb + tid] = 0.f;
    return;
  }
  int k0 = 0, k1 = 0;
  if (tile.seq >= 0) {
    k0 = min(max(a.k_ptr[tile.seq], 0), a.Nk);
    k1 = min(max(a.k_ptr[tile.seq + 1], k0), a.Nk);
  }
  const T* q = (const T*)a.q + h * a.q_head;
  const T* dout = (const T*)a.d_out + h * a.do_head;
  const T* k = (const T*)a.k + (h / a.G) * a.k_head;
  const T* v = (const T*)a.v + (h / a.G) * a.v_head;

  const int r0 = tile.start + wave * 16 * NQ;
  const bool active = r0 < tile.end;
  typename M::Row qf[NQ], df[NQ];
  Pos qp[NQ];
  f4 dq[NQ][M::DT];
  float lse[NQ], delta[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int row = r0 + 16 * n + li;
    const bool ok = row < tile.end;
    qf[n] = M::row_global(q + (int64_t)row * a.q_row, g, a.D, ok, a.vec_q);
    df[n] = M::row_global(dout + (int64_t)row * a.do_row, g, a.D, ok, a.vec_do);
    qp[n] = load_pos<BIAS>(a.q_pos, row, ok);
    const bool vec_o = a.D % El<T>::kPer == 0;
    const typename M::Row of = M::row_global((const T*)a.out + ((int64_t)row * a.H + h) * a.D, g, a.D, ok, vec_o);
    // the diagonal of O dO^T, by the very products that give dP: a row with one key has o = v, so its
    // dP - delta is zero and not the rounding of two orders of one sum
    f4 od = M::dot(of, df[n], f4{0.f, 0.f, 0.f, 0.f});
    if (a.rest != nullptr)
      od = M::dot(M::row_global((const T*)a.rest + ((int64_t)row * a.H + h) * a.D, g, a.D, ok, vec_o), df[n], od);
    float mine = 0.f;
#pragma unroll
    for (int r = 0; r < 4; ++r) mine = li == 4 * g + r ? od[r] : mine;
    delta[n] = column_sum(mine);
    lse[n] = ok ? a.lse[(int64_t)h * a.Nq + row] : INFINITY;  // exp2(z - inf): a row that is not there has no p
    if (ok && g == 0) a.delta[(int64_t)h * a.Nq + row] = delta[n];
#pragma unroll
    for (int d = 0; d < M::DT; ++d) dq[n][d] = f4{0.f, 0.f, 0.f, 0.f};
  }
  if constexpr (BIAS != kNoBias) {
    const float* tab = (const float*)a.table + h * nb;
    for (int i = tid; i < nl; i += 256) {
      const int b = lut_bucket<BIAS>(a.rule, i);
      lut[i] = tab[b] * kLog2e;
      lutb[i] = (uint8_t)b;
    }
    for (int i = tid; i < 4 * nb * 64; i += 256) hist[i] = 0.f;
  }
  const float c = a.scale * kLog2e;

  Stage<T, DP> sk, sv;
  if (k0 < k1) {
    sk.load(k, a.k_row, k0, k1, a.key_mask, a.D, a.vec_k, tid);
    sv.load(v, a.v_row, k0, k1, a.key_mask, a.D, a.vec_v, tid);
  }
  for (int kt = k0; kt < k1; kt += kTile) {
    __syncthreads();
    sk.store(Ks, tid);
    sv.store(Vs, tid);
    if (tid < kTile) {
      const int row = kt + tid;
      kadd[tid] = row < k1 && (a.key_mask == nullptr || a.key_mask[row] != 0) ? 0.f : -INFINITY;
    }
    stage_pos<BIAS>(kpos, a.k_pos, kt, k1, tid);
    __syncthreads();
    if (kt + kTile < k1) {
      sk.load(k, a.k_row, kt + kTile, k1, a.key_mask, a.D, a.vec_k, tid);
      sv.load(v, a.v_row, kt + kTile, k1, a.key_mask, a.D, a.vec_v, tid);
    }
    if (!active) continue;
    const bool some = a.key_mask != nullptr || kt + kTile > k1;
#pragma unroll
    for (int u = 0; u < kTile / 32; ++u) {
      f4 ds[2][NQ];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int at = 32 * u + 16 * t;
        const typename M::Row kf = M::row_lds(Ks + (at + li) * M::LD, g);
        const typename M::Row vf = M::row_lds(Vs + (at + li) * M::LD, g);
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          f4 x = M::dot(kf, qf[n], f4{0.f, 0.f, 0.f, 0.f}) * c;
          const f4 dp = M::dot(vf, df[n], f4{0.f, 0.f, 0.f, 0.f});
          int e[4];
          if constexpr (BIAS == kOrder) {
            const int4 kp = *reinterpret_cast<const int4*>(kpos + at + 4 * g);
            e[0] = order_index(kp.x, qp[n].i, a.rule.far);
            e[1] = order_index(kp.y, qp[n].i, a.rule.far);
            e[2] = order_index(kp.z, qp[n].i, a.rule.far);
            e[3] = order_index(kp.w, qp[n].i, a.rule.far);
          } else if constexpr (BIAS == kSpace) {
            const float* kp = (const float*)kpos + at + 4 * g;
            const f4 kx = *(const f4*)kp, ky = *(const f4*)(kp + kTile), kz = *(const f4*)(kp + 2 * kTile);
#pragma unroll
            for (int r = 0; r < 4; ++r)
              e[r] = space_index(qp[n].x, qp[n].y, qp[n].z, kx[r], ky[r], kz[r], a.rule);
          }
          if constexpr (BIAS != kNoBias) {
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] += lut[e[r]];
          }
          if (some) x += *reinterpret_cast<const f4*>(kadd + at + 4 * g);
#pragma unroll
          for (int r = 0; r < 4; ++r) ds[t][n][r] = __builtin_amdgcn_exp2f(x[r] - lse[n]) * (dp[r] - delta[n]);
          if constexpr (BIAS != kNoBias) {
#pragma unroll
            for (int r = 0; r < 4; ++r) hist[(wave * nb + lutb[e[r]]) * 64 + lane] += ds[t][n][r];
          }
        }
      }
      M::template outer<NQ, false>(Ks + 32 * u * M::LD, ds[0], ds[1], dq, lane);
    }
  }
  if (active) {
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int row = r0 + 16 * n + li;
      if (row < tile.end) M::store((T*)a.dq + ((int64_t)row * a.H + h) * a.D, dq[n], a.scale, a.D, g);
    }
  }
  if constexpr (BIAS != kNoBias) {
    __syncthreads();
    for (int b = wave; b < nb; b += 4) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) t += hist[(w * nb + b) * 64 + lane];
      t = wave_sum(t);
      if (lane == 0) a.part[(int64_t)blockIdx.x * nb + b] = t;
    }
  }
}

// The table's gradient: one wave adds the tiles' sums of one (head, bucket), in 64 bits and in order.
__global__ __launch_bounds__(64) void bwd_table_kernel(const float* part, float* out, int tiles, int cells) {
  const int cell = blockIdx.x, lane = threadIdx.x;
  double t = 0.0;
  for (int i = lane; i < tiles; i += 64) t += (double)part[(int64_t)i * cells + cell];
  t = wave_sum(t);
  if (lane == 0) out[cell] = (float)t;
}

// ------------------------------------------------------------------ key pass
template <typename T, int DP, int NK, int BIAS>
__global__ __launch_bounds__(256) void bwd_key_kernel(Args a) {
  typedef Mat<T, DP> M;
  constexpr int ROWS = 64 * NK;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  T* Qs = (T*)smem;
  T* Ds = Qs + kTile * M::LD;
  float* qlse = (float*)(Ds + kTile * M::LD);
  float* qdel = qlse + kTile;
  int* qpos = (int*)(qdel + kTile);
  float* lut = (float*)(qpos + 3 * kTile);

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, li = lane & 15;
  const int hk = blockIdx.x % a.Hk;
  const Tile tile = find_tile(a.k_ptr, a.S, a.Nk, ROWS, blockIdx.x / a.Hk);
  if (tile.start >= tile.end) return;
  int q0 = 0, q1 = 0;
  if (tile.seq >= 0) {
    q0 = min(max(a.q_ptr[tile.seq], 0), a.Nq);
    q1 = min(max(a.q_ptr[tile.seq + 1], q0), a.Nq);
  }
  const T* k = (const T*)a.k + hk * a.k_head;
  const T* v = (const T*)a.v + hk * a.v_head;
  const int r0 = tile.start + wave * 16 * NK;
  const bool active = r0 < tile.end;
  typename M::Row kf[NK], vf[NK];
  Pos kp[NK];
  bool keep[NK];
  f4 dk[NK][M::DT], dv[NK][M::DT];
#pragma unroll
  for (int n = 0; n < NK; ++n) {
    const int row = r0 + 16 * n + li;
    const bool ok = row < tile.end;
    keep[n] = ok && (a.key_mask == nullptr || a.key_mask[row] != 0);
    kf[n] = M::row_global(k + (int64_t)row * a.k_row, g, a.D, keep[n], a.vec_k);
    vf[n] = M::row_global(v + (int64_t)row * a.v_row, g, a.D, keep[n], a.vec_v);
    kp[n] = load_pos<BIAS>(a.k_pos, row, ok);
#pragma unroll
    for (int d = 0; d < M::DT; ++d) dk[n][d] = dv[n][d] = f4{0.f, 0.f, 0.f, 0.f};
  }
  const float c = a.scale * kLog2e;
  for (int h = hk * a.G; h < (hk + 1) * a.G; ++h) {
    const T* q = (const T*)a.q + h * a.q_head;
    const T* dout = (const T*)a.d_out + h * a.do_head;
    Stage<T, DP> sq, sd;
    if (q0 < q1) {
      sq.load(q, a.q_row, q0, q1, nullptr, a.D, a.vec_q, tid);
      sd.load(dout, a.do_row, q0, q1, nullptr, a.D, a.vec_do, tid);
    }
    if constexpr (BIAS != kNoBias) {
      __syncthreads();  // the head before is done with the look-up table
      const float* tab = (const float*)a.table + h * a.rule.buckets;
      for (int i = tid; i < lut_size<BIAS>(a.rule); i += 256) lut[i] = tab[lut_bucket<BIAS>(a.rule, i)] * kLog2e;
    }
    for (int qt = q0; qt < q1; qt += kTile) {
      __syncthreads();
      sq.store(Qs, tid);
      sd.store(Ds, tid);
      if (tid < kTile) {
        const int row = qt + tid;
        qlse[tid] = row < q1 ? a.lse[(int64_t)h * a.Nq + row] : INFINITY;
        qdel[tid] = row < q1 ? a.delta[(int64_t)h * a.Nq + row] : 0.f;
      }
      stage_pos<BIAS>(qpos, a.q_pos, qt, q1, tid);
      __syncthreads();
      if (qt + kTile < q1) {
        sq.load(q, a.q_row, qt + kTile, q1, nullptr, a.D, a.vec_q, tid);
        sd.load(dout, a.do_row, qt + kTile, q1, nullptr, a.D, a.vec_do, tid);
      }
      if (!active) continue;
#pragma unroll
      for (int u = 0; u < kTile / 32; ++u) {
        f4 p[2][NK], ds[2][NK];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int at = 32 * u + 16 * t;
          const typename M::Row qf = M::row_lds(Qs + (at + li) * M::LD, g);
          const typename M::Row df = M::row_lds(Ds + (at + li) * M::LD, g);
          const f4 lse = *reinterpret_cast<const f4*>(qlse + at + 4 * g);
          const f4 del = *reinterpret_cast<const f4*>(qdel + at + 4 * g);
#pragma unroll
          for (int n = 0; n < NK; ++n) {
            f4 x = M::dot(qf, kf[n], f4{0.f, 0.f, 0.f, 0.f}) * c;
            const f4 dp = M::dot(df, vf[n], f4{0.f, 0.f, 0.f, 0.f});
            if constexpr (BIAS == kOrder) {
              const int4 qp = *reinterpret_cast<const int4*>(qpos + at + 4 * g);
              x[0] += lut[order_index(kp[n].i, qp.x, a.rule.far)];
              x[1] += lut[order_index(kp[n].i, qp.y, a.rule.far)];
              x[2] += lut[order_index(kp[n].i, qp.z, a.rule.far)];
              x[3] += lut[order_index(kp[n].i, qp.w, a.rule.far)];
            } else if constexpr (BIAS == kSpace) {
              const float* qp = (const float*)qpos + at + 4 * g;
              const f4 qx = *(const f4*)qp, qy = *(const f4*)(qp + kTile), qz = *(const f4*)(qp + 2 * kTile);
#pragma unroll
              for (int r = 0; r < 4; ++r)
                x[r] += lut[space_index(qx[r], qy[r], qz[r], kp[n].x, kp[n].y, kp[n].z, a.rule)];
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float e = keep[n] ? __builtin_amdgcn_exp2f(x[r] - lse[r]) : 0.f;
              p[t][n][r] = e;
              ds[t][n][r] = e * (dp[r] - del[r]);
            }
          }
        }
        M::template outer<NK, false>(Ds + 32 * u * M::LD, p[0], p[1], dv, lane);
        M::template outer<NK, false>(Qs + 32 * u * M::LD, ds[0], ds[1], dk, lane);
      }
    }
  }
  if (!active) return;
#pragma unroll
  for (int n = 0; n < NK; ++n) {
    const int row = r0 + 16 * n + li;
    if (row < tile.end) {
      M::store((T*)a.dk + ((int64_t)row * a.Hk + hk) * a.D, dk[n], a.scale, a.D, g);
      M::store((T*)a.dv + ((int64_t)row * a.Hk + hk) * a.D, dv[n], 1.f, a.D, g);
    }
  }
}

static int query_rows(at::ScalarType t) { return t == at::kFloat ? 64 : 128; }

int64_t table_tiles(int64_t Nq, int64_t S, at::ScalarType t) { return tile_count(Nq, S, query_rows(t)); }

template <typename F>
static void allow_lds(F* kern, size_t lds) {
  if (lds > 65536) (void)hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
}

template <typename T, int DP, int NQ, int BIAS>
static void launch_bwd(const Args& a, float* dtable, hipStream_t st) {
  const size_t tiles2 = 2 * kTile * Mat<T, DP>::LD * sizeof(T);
  const int nl = BIAS == kOrder ? 2 * a.rule.far + 1 : BIAS == kSpace ? a.rule.far + 1 : 0;
  const int64_t qt = tile_count(a.Nq, a.S, 64 * NQ), kt = tile_count(a.Nk, a.S, 64 * NQ);
  HY_CHECK(qt * a.H < (int64_t(1) << 31) && kt * a.Hk < (int64_t(1) << 31),
           "cross_attention: too many tiles for one launch");
  {
    size_t lds = tiles2 + 4 * kTile * 4;
    if (BIAS != kNoBias) lds += 4 * a.rule.buckets * 64 * 4 + nl * 5;
    auto* kern = &bwd_query_kernel<T, DP, NQ, BIAS>;
    allow_lds(kern, lds);
    kern<<<dim3((unsigned)(qt * a.H)), 256, lds, st>>>(a);
  }
  if (BIAS != kNoBias) {
    const int cells = a.H * a.rule.buckets;
    bwd_table_kernel<<<dim3(cells), 64, 0, st>>>(a.part, dtable, (int)qt, cells);
  }
  {
    const size_t lds = tiles2 + 5 * kTile * 4 + nl * 4;
    auto* kern = &bwd_key_kernel<T, DP, NQ, BIAS>;
    allow_lds(kern, lds);
    kern<<<dim3((unsigned)(kt * a.Hk)), 256, lds, st>>>(a);
  }
}

template <typename T, int DP, int NQ>
static void pick_bias(const Args& a, int bias, float* dtable, hipStream_t st) {
  if (bias == kNoBias) launch_bwd<T, DP, NQ, kNoBias>(a, dtable, st);
  else if (bias == kOrder) launch_bwd<T, DP, NQ, kOrder>(a, dtable, st);
  else launch_bwd<T, DP, NQ, kSpace>(a, dtable, st);
}

void backward(const Args& a, at::ScalarType t, int bias, float* dtable, hipStream_t st) {
  if (t == at::kFloat) {
    if (a.D <= 16) pick_bias<float, 16, 1>(a, bias, dtable, st);
    else if (a.D <= 32) pick_bias<float, 32, 1>(a, bias, dtable, st);
    else if (a.D <= 64) pick_bias<float, 64, 1>(a, bias, dtable, st);
    else pick_bias<float, 128, 1>(a, bias, dtable, st);
  } else if (t == at::kBFloat16) {
    if (a.D <= 32) pick_bias<__bf16, 32, 2>(a, bias, dtable, st);
    else if (a.D <= 64) pick_bias<__bf16, 64, 2>(a, bias, dtable, st);
    else pick_bias<__bf16, 128, 2>(a, bias, dtable, st);
  } else {
    if (a.D <= 32) pick_bias<_Float16, 32, 2>(a, bias, dtable, st);
    else if (a.D <= 64) pick_bias<_Float16, 64, 2>(a, bias, dtable, st);
    else pick_bias<_Float16, 128, 2>(a, bias, dtable, st);
  }
}

}  // namespace xa
}  // namespace hy
