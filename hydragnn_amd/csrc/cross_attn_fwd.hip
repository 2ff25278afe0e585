// Ragged cross attention, forward (see cross_attn.h for the mathematics and the layouts).
//
// A workgroup owns 64 NQ query rows of one sequence and one head; each of its four waves owns
// 16 NQ of them and streams over all keys, whose tiles of 64 the workgroup stages in LDS once.
#include "cross_attn.h"

namespace hy {
namespace xa {

template <typename T, int DP, int NQ, int BIAS, bool SAVE, bool VEC>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(DP > 64 ? 2 : 3))) void fwd_kernel(Args a) {
  typedef Mat<T, DP> M;
  typedef Tiles<T, DP, 1> L;
  constexpr int ROWS = 64 * NQ, TK = L::TK, KB = TK / 16;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  float* lut = (float*)(smem + 2 * L::kBytes);

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, li = lane & 15;
  const int h = blockIdx.x % a.H;
  const Tile tile = find_tile(a.q_ptr, a.S, a.Nq, ROWS, blockIdx.x / a.H);
  if (tile.start >= tile.end) return;
  int k0 = 0, k1 = 0;
  if (tile.seq >= 0) {
    k0 = min(max(a.k_ptr[tile.seq], 0), a.Nk);
    k1 = min(max(a.k_ptr[tile.seq + 1], k0), a.Nk);
  }
  const T* k = (const T*)a.k + (h / a.G) * a.k_head;
  const T* v = (const T*)a.v + (h / a.G) * a.v_head;

  const int r0 = wave * 16 * NQ, rows = tile.end - tile.start;  // of the tile
  const bool active = r0 < rows;
  typename M::Row qf[NQ];
  float c = 1.f;
  Pos qp[NQ];
  Span span = {INT_MAX, INT_MIN};
  f4 o[NQ][M::DT];
  float m[NQ], l[NQ];
  {
    const Rsrc rq = rsrc_of((const T*)a.q + h * a.q_head + (int64_t)tile.start * a.q_row);
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int row = r0 + 16 * n + li;
      const bool ok = row < rows;
      qf[n] = M::row_global(rq, row * (int)(a.q_row * sizeof(T)), g, a.D, ok, a.unit_q);
      c = M::take_scale(qf[n], a.scale);
      qp[n] = load_pos<BIAS>(a.q_pos, tile.start + row, ok);
      if (BIAS == kOrder) {
        span.lo = min(span.lo, wave_min_i32(ok ? qp[n].i : INT_MAX));
        span.hi = max(span.hi, wave_max_i32(ok ? qp[n].i : INT_MIN));
      }
      m[n] = -INFINITY;
      l[n] = 0.f;
#pragma unroll
      for (int d = 0; d < M::DT; ++d) o[n][d] = f4{0.f, 0.f, 0.f, 0.f};
    }
  }
  if constexpr (BIAS != kNoBias) {
    const float* tab = (const float*)a.table + h * a.rule.buckets;
    for (int i = tid; i < lut_size<BIAS>(a.rule); i += 256) lut[i] = tab[lut_bucket<BIAS>(a.rule, i)] * kLog2e;
  }

  // s is an exponent of 2 where the scale or a bias is in it, else a product that c makes one
  constexpr bool kDone = M::kScaled || BIAS != kNoBias;
  auto power = [&](float s, float top) {
    return __builtin_amdgcn_exp2f(kDone ? s - top : fmaf(s, c, -top * c));
  };

  typedef Stage<T, DP, VEC> St;
  St sk, sv;
  typename St::Keep keep;
  sk.init(a.k_row, a.D, tid);
  sv.init(a.v_row, a.D, tid);
  StagePos<BIAS, TK> sp;
  auto fetch = [&](int kt) {  // a tile's rows, with the masks that the call before has fetched
    sk.load(k, a.k_row, kt, k1 - kt, keep, a.D, a.unit_k, tid);
    sv.load(v, a.v_row, kt, k1 - kt, keep, a.D, a.unit_v, tid);
    sp.load(a.k_pos, kt, k1 - kt, tid);
  };
  float add = 0.f;
  auto masks = [&](int kt) {
    St::keep(keep, a.key_mask, kt, k1 - kt, tid);
    add = key_flag(a.key_mask, kt, k1 - kt, tid & (TK - 1));
  };
  auto put = [&](int buf, int kt, float flag) {
    const L t(smem, buf);
    sk.store(t.a, tid);
    sv.store(t.b, tid);
    sp.store(t.pos, k1 - kt, tid);
    if (tid < TK) t.f[tid] = flag;
  };
  if (k0 < k1) {
    masks(k0);
    fetch(k0);
    put(0, k0, add);
    masks(min(k0 + TK, k1));
  }
  int buf = 0;
  for (int kt = k0; kt < k1; kt += TK, buf ^= 1) {
    __syncthreads();  // this tile is there, and every wave is done with the one before it
    const bool more = kt + TK < k1;
    const float flag = add;
    if (more) {
      fetch(kt + TK);
      masks(min(kt + 2 * TK, k1));
    }
    const L t(smem, buf);
    if (active) {
      f4 s[KB][NQ];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {  // a key's 0 or -inf is what its products are added to
        const typename M::Row kf = M::row_lds(t.a + (16 * kb + li) * M::LD, g);
        const f4 off = *reinterpret_cast<const f4*>(t.f + 16 * kb + 4 * g);
#pragma unroll
        for (int n = 0; n < NQ; ++n) s[kb][n] = M::dot(kf, qf[n], off);
      }
      if constexpr (BIAS != kNoBias) {
        const int one = BIAS == kOrder ? far_entry(t.span(), span, a.rule.far) : -1;
        if (one >= 0) {
          const float b = lut[one];
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
              for (int r = 0; r < 4; ++r) s[kb][n][r] = fmaf(s[kb][n][r], c, b);
        } else {
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
              const Index<BIAS, TK> e(t.pos, 16 * kb + 4 * g, qp[n], a.rule);
#pragma unroll
              for (int r = 0; r < 4; ++r) s[kb][n][r] = fmaf(s[kb][n][r], c, lut[e.i[r]]);
            }
        }
      }
      float shrink[NQ];
      bool grown = false;
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        float top = m[n];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
          top = fmaxf(fmaxf(fmaxf(fmaxf(top, s[kb][n][0]), s[kb][n][1]), s[kb][n][2]), s[kb][n][3]);
        top = column_max(top);
        const float at = top == -INFINITY ? 0.f : top;  // no key so far: every p is exp2(-inf)
        shrink[n] = power(m[n], at);
        grown |= top > m[n];
        m[n] = top;
        float sum = 0.f;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            s[kb][n][r] = power(s[kb][n][r], at);
            sum += s[kb][n][r];
          }
        // of this lane's keys; the four lanes of a row are joined at the end.  (m = -inf: l is 0.)
        l[n] = fmaf(l[n], shrink[n], sum);
      }
      if (__any(grown)) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          float by = shrink[n];
          asm volatile("" : "+v"(by));  // (keeps the products inside the branch, which few tiles take)
#pragma unroll
          for (int d = 0; d < M::DT; ++d) o[n][d] *= by;
        }
      }
#pragma unroll
      for (int u = 0; u < TK / 32; ++u)
        M::template outer<NQ, SAVE>(t.b + 32 * u * M::LD, s[2 * u], s[2 * u + 1], o, lane);
    }
    if (more) put(buf ^ 1, kt + TK, flag);
  }
  if (!active) return;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int row = tile.start + r0 + 16 * n + li;
    const float sum = column_sum(l[n]);
    if (row < tile.end) {
      const int64_t at = ((int64_t)row * a.H + h) * a.D;
      M::store((T*)a.out + at, o[n], sum > 0.f || sum != sum ? 1.f / sum : 0.f, a.D, g,
               SAVE ? (T*)a.rest + at : nullptr);
      if (SAVE && g == 0)
        a.lse[(int64_t)h * a.Nq + row] =
            m[n] == -INFINITY ? INFINITY : (kDone ? m[n] : m[n] * c) + __builtin_amdgcn_logf(sum);
    }
  }
}

template <typename T, int DP, int NQ, int BIAS>
static void launch_fwd(const Args& a, hipStream_t st) {
  const int64_t blocks = tile_count(a.Nq, a.S, 64 * NQ) * a.H;
  HY_CHECK(blocks < (int64_t(1) << 31), "cross_attention: too many query tiles for one launch");
  size_t lds = 2 * Tiles<T, DP, 1>::kBytes;
  if (BIAS == kOrder) lds += (2 * a.rule.far + 1) * 4;
  if (BIAS == kSpace) lds += (a.rule.far + 1) * 4;
  const bool vec = a.unit_k == 16 && a.unit_v == 16;
  auto* kern = a.lse != nullptr
                   ? (vec ? &fwd_kernel<T, DP, NQ, BIAS, true, true> : &fwd_kernel<T, DP, NQ, BIAS, true, false>)
                   : (vec ? &fwd_kernel<T, DP, NQ, BIAS, false, true> : &fwd_kernel<T, DP, NQ, BIAS, false, false>);
  allow_lds((const void*)kern, lds);
  kern<<<dim3((unsigned)blocks), 256, lds, st>>>(a);
}

// 16 bits: 32 rows a wave, so that a key fragment read from LDS feeds two products, where that leaves
// eight workgroups a compute unit to even out sequences of unlike length; else 16, as with distances,
// whose arithmetic wants the registers.
template <typename T, int DP>
static void pick(const Args& a, int bias, hipStream_t st) {
  constexpr int N2 = sizeof(T) == 2 ? 2 : 1;
  const bool two = N2 == 2 && (int64_t)(a.Nq / 128) * a.H >= 8 * num_cus();
  if (bias == kNoBias) two ? launch_fwd<T, DP, N2, kNoBias>(a, st) : launch_fwd<T, DP, 1, kNoBias>(a, st);
  else if (bias == kOrder) two ? launch_fwd<T, DP, N2, kOrder>(a, st) : launch_fwd<T, DP, 1, kOrder>(a, st);
  else launch_fwd<T, DP, 1, kSpace>(a, st);
}

template <typename T>
static void pick_width(const Args& a, int bias, hipStream_t st) {
  if (sizeof(T) == 4 && a.D <= 16) pick<T, sizeof(T) == 4 ? 16 : 32>(a, bias, st);
  else if (a.D <= 32) pick<T, 32>(a, bias, st);
  else if (a.D <= 64) pick<T, 64>(a, bias, st);
  else pick<T, 128>(a, bias, st);
}

void forward(const Args& a, at::ScalarType t, int bias, hipStream_t st) {
  if (t == at::kFloat) pick_width<float>(a, bias, st);
  else if (t == at::kBFloat16) pick_width<__bf16>(a, bias, st);
  else pick_width<_Float16>(a, bias, st);
}

}  // namespace xa
}  // namespace hy
