// Ragged cross attention, forward (see cross_attn.h for the mathematics and the layouts).
//
// A workgroup owns 64 NQ query rows of one sequence and one head; each of its four waves owns
// 16 NQ of them and streams over all keys, whose tiles of 64 the workgroup stages in LDS once.
#include "cross_attn.h"

namespace hy {
namespace xa {

template <typename T, int DP, int NQ, int BIAS, bool SAVE>
__global__ __launch_bounds__(256) void fwd_kernel(Args a) {
  typedef Mat<T, DP> M;
  constexpr int ROWS = 64 * NQ;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  T* Ks = (T*)smem;
  T* Vs = Ks + kTile * M::LD;
  float* kadd = (float*)(Vs + kTile * M::LD);  // 0, or -inf where the key takes no part
  int* kpos = (int*)(kadd + kTile);
  float* lut = (float*)(kpos + 3 * kTile);

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, li = lane & 15;
  const int h = blockIdx.x % a.H;
  const Tile tile = find_tile(a.q_ptr, a.S, a.Nq, ROWS, blockIdx.x / a.H);
  if (tile.start >= tile.end) return;
  int k0 = 0, k1 = 0;
  if (tile.seq >= 0) {
    k0 = min(max(a.k_ptr[tile.seq], 0), a.Nk);
    k1 = min(max(a.k_ptr[tile.seq + 1], k0), a.Nk);
  }
  const T* q = (const T*)a.q + h * a.q_head;
  const T* k = (const T*)a.k + (h / a.G) * a.k_head;
  const T* v = (const T*)a.v + (h / a.G) * a.v_head;

  const int r0 = tile.start + wave * 16 * NQ;
  const bool active = r0 < tile.end;
  typename M::Row qf[NQ];
  Pos qp[NQ];
  f4 o[NQ][M::DT];
  float m[NQ], l[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int row = r0 + 16 * n + li;
    const bool ok = row < tile.end;
    qf[n] = M::row_global(q + (int64_t)row * a.q_row, g, a.D, ok, a.vec_q);
    qp[n] = load_pos<BIAS>(a.q_pos, row, ok);
    m[n] = -INFINITY;
    l[n] = 0.f;
#pragma unroll
    for (int d = 0; d < M::DT; ++d) o[n][d] = f4{0.f, 0.f, 0.f, 0.f};
  }
  if constexpr (BIAS != kNoBias) {
    const float* tab = (const float*)a.table + h * a.rule.buckets;
    for (int i = tid; i < lut_size<BIAS>(a.rule); i += 256) lut[i] = tab[lut_bucket<BIAS>(a.rule, i)] * kLog2e;
  }
  const float c = a.scale * kLog2e;

  Stage<T, DP> sk, sv;
  if (k0 < k1) {
    sk.load(k, a.k_row, k0, k1, a.key_mask, a.D, a.vec_k, tid);
    sv.load(v, a.v_row, k0, k1, a.key_mask, a.D, a.vec_v, tid);
  }
  for (int kt = k0; kt < k1; kt += kTile) {
    __syncthreads();  // the tile before is done with
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
    f4 s[kTile / 16][NQ];
#pragma unroll
    for (int kb = 0; kb < kTile / 16; ++kb) {
      const typename M::Row kf = M::row_lds(Ks + (16 * kb + li) * M::LD, g);
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        f4 x = M::dot(kf, qf[n], f4{0.f, 0.f, 0.f, 0.f}) * c;
        if constexpr (BIAS == kOrder) {
          const int4 kp = *reinterpret_cast<const int4*>(kpos + 16 * kb + 4 * g);
          x[0] += lut[order_index(kp.x, qp[n].i, a.rule.far)];
          x[1] += lut[order_index(kp.y, qp[n].i, a.rule.far)];
          x[2] += lut[order_index(kp.z, qp[n].i, a.rule.far)];
          x[3] += lut[order_index(kp.w, qp[n].i, a.rule.far)];
        } else if constexpr (BIAS == kSpace) {
          const float* kp = (const float*)kpos + 16 * kb + 4 * g;
          const f4 kx = *(const f4*)kp, ky = *(const f4*)(kp + kTile), kz = *(const f4*)(kp + 2 * kTile);
#pragma unroll
          for (int r = 0; r < 4; ++r)
            x[r] += lut[space_index(qp[n].x, qp[n].y, qp[n].z, kx[r], ky[r], kz[r], a.rule)];
        }
        if (some) x += *reinterpret_cast<const f4*>(kadd + 16 * kb + 4 * g);
        s[kb][n] = x;
      }
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float top = m[n];
#pragma unroll
      for (int kb = 0; kb < kTile / 16; ++kb)
        top = fmaxf(top, fmaxf(fmaxf(s[kb][n][0], s[kb][n][1]), fmaxf(s[kb][n][2], s[kb][n][3])));
      top = column_max(top);
      const float at = top == -INFINITY ? 0.f : top;  // no key so far: every p is exp2(-inf)
      if (__any(top > m[n])) {
        const float shrink = __builtin_amdgcn_exp2f(m[n] - at);
        l[n] *= shrink;
#pragma unroll
        for (int d = 0; d < M::DT; ++d) o[n][d] *= shrink;
      }
      m[n] = top;
      float sum = 0.f;
#pragma unroll
      for (int kb = 0; kb < kTile / 16; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[kb][n][r] = __builtin_amdgcn_exp2f(s[kb][n][r] - at);
          sum += s[kb][n][r];
        }
      l[n] += sum;  // of this lane's keys; the four lanes of a row are joined at the end
    }
#pragma unroll
    for (int u = 0; u < kTile / 32; ++u) 
      M::template outer<NQ, SAVE>(Vs + 32 * u * M::LD, s[2 * u], s[2 * u + 1], o, lane);
  }
  if (!active) return;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int row = r0 + 16 * n + li;
    const float sum = column_sum(l[n]);
    if (row < tile.end) {
      const int64_t at = ((int64_t)row * a.H + h) * a.D;
      M::store((T*)a.out + at, o[n], sum > 0.f || sum != sum ? 1.f / sum : 0.f, a.D, g,
               SAVE ? (T*)a.rest + at : nullptr);
      if (SAVE && g == 0)
        a.lse[(int64_t)h * a.Nq + row] = m[n] == -INFINITY ? INFINITY : m[n] + __builtin_amdgcn_logf(sum);
    }
  }
}

template <typename T, int DP, int NQ, int BIAS>
static void launch_fwd(const Args& a, hipStream_t st) {
  const int64_t blocks = tile_count(a.Nq, a.S, 64 * NQ) * a.H;
  HY_CHECK(blocks < (int64_t(1) << 31), "cross_attention: too many query tiles for one launch");
  size_t lds = 2 * kTile * Mat<T, DP>::LD * sizeof(T) + 4 * kTile * 4;
  if (BIAS == kOrder) lds += (2 * a.rule.far + 1) * 4;
  if (BIAS == kSpace) lds += (a.rule.far + 1) * 4;
  auto* kern = a.lse != nullptr ? &fwd_kernel<T, DP, NQ, BIAS, true> : &fwd_kernel<T, DP, NQ, BIAS, false>;
  if (lds > 65536) (void)hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  kern<<<dim3((unsigned)blocks), 256, lds, st>>>(a);
}

template <typename T, int DP, int NQ>
static void pick_bias(const Args& a, int bias, hipStream_t st) {
  if (bias == kNoBias) launch_fwd<T, DP, NQ, kNoBias>(a, st);
  else if (bias == kOrder) launch_fwd<T, DP, NQ, kOrder>(a, st);
  else launch_fwd<T, DP, NQ, kSpace>(a, st);
}

void forward(const Args& a, at::ScalarType t, int bias, hipStream_t st) {
  if (t == at::kFloat) {
    if (a.D <= 16) pick_bias<float, 16, 1>(a, bias, st);
    else if (a.D <= 32) pick_bias<float, 32, 1>(a, bias, st);
    else if (a.D <= 64) pick_bias<float, 64, 1>(a, bias, st);
    else pick_bias<float, 128, 1>(a, bias, st);
  } else if (t == at::kBFloat16) {
    if (a.D <= 32) pick_bias<__bf16, 32, 2>(a, bias, st);
    else if (a.D <= 64) pick_bias<__bf16, 64, 2>(a, bias, st);
    else pick_bias<__bf16, 128, 2>(a, bias, st);
  } else {
    if (a.D <= 32) pick_bias<_Float16, 32, 2>(a, bias, st);
    else if (a.D <= 64) pick_bias<_Float16, 64, 2>(a, bias, st);
    else pick_bias<_Float16, 128, 2>(a, bias, st);
  }
}

}  // namespace xa
}  // namespace hy
