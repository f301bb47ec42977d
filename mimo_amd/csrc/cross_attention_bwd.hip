// cross_attention_bwd.hip — gradients of the cross attention (gfx950, MFMA 32x32x16).
//
//   P = exp(scale q.k - lse), delta[q] = sum_d dO o O, dP = dO.V^T, dS = P (dP - delta)
//   dQ = scale dS.K          dK = scale dS^T.Q          dV = P^T.dO        (dK, dV: summed over every query that sees the key)
//
// Two kernels, both recompute P from lse (no score is ever stored):
//   xattn_dq_kernel   S^T = K.Q^T and dP^T = V.dO^T: a lane owns a query, dS^T packed is the operand of dQ^T = K^T.dS^T.  Keys
//                     resident in LDS as in the forward, or streamed; also leaves delta.
//   xattn_dkv_kernel  S = Q.K^T and dP = dO.V^T: a lane owns a key, a wave 32 of them with K and V in registers; the block's waves
//                     share the query tiles that pass through LDS, P and dS packed are the operands of dV^T = dO^T.P and
//                     dK^T = Q^T.dS.  The flat rows are cut into parts (gridDim.y) when the keys do not fill the chip; their
//                     fp32 sums are joined in a fixed order by xattn_dkv_join_kernel: no atomics, the same bits every time.
// P and dS are rounded to the operand type for the last products (one rounding each of the size of the results' own); sums, lse
// and delta are fp32.
#include "cross_attention.hip.h"

namespace mimo_xattn {
namespace {

constexpr int CH = 64;
constexpr int RES_LDS = 80000;

template <int DT, int KS, bool RESIDENT>
__global__ __launch_bounds__(256, KS <= 3 ? 3 : KS <= 6 ? 2 : 1) void xattn_dq_kernel(const Args a) {
  constexpr int OT = (KS + 1) / 2, P = 16 * KS + 8, THREADS = 256;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h2 = lane >> 5, li = lane & 31;
  const unsigned L = xcd_remap(blockIdx.x, gridDim.x);
  const int g = (int)(L % (unsigned)a.kvh);
  const int j = (int)(L / (unsigned)a.kvh) % a.nb, e = (int)(L / (unsigned)a.kvh) / a.nb;
  const int len = valid_len(a, e);
  const int T = (a.R + 31) >> 5;
  const int npad = RESIDENT ? (a.Nk + 31) / 32 * 32 : CH;
  uint16_t* const ks = reinterpret_cast<uint16_t*>(smem);
  uint16_t* const vs = ks + npad * P;
  float* const bias = reinterpret_cast<float*>(smem + 2 * npad * P * 2 + 64);
  if constexpr (RESIDENT) {
    stage_kv<KS, THREADS>(a, e, g, len, 0, (len + 31) / 32 * 32, ks, vs, bias, tid);
    __syncthreads();
  }
  const int step = a.nb * 4;
  int t = j * 4 + wave;
  const int rounds = (T - j * 4 + step - 1) / step;

  for (int round = 0; RESIDENT ? t < T : round < rounds; t += step, ++round) {
    const int f = 32 * t + li;
    const bool live = f < a.R;
    int img, qi, hh;
    flat_row(a, min(f, a.R - 1), img, qi, hh);
    const int head = g * a.hg + hh;
    const int64_t b = (int64_t)e * a.G + img, col = (int64_t)head * a.d;
    const int64_t stat = (b * a.kvh * a.hg + head) * a.Nq + qi;
    uint4 qf[KS], df[KS];
    load_row<KS>(qf, a.q + b * a.sqb + (int64_t)qi * a.sqr + col, a.d, h2);
    load_row<KS>(df, a.dout + b * a.sdb + (int64_t)qi * a.sdr + col, a.d, h2);
    float delta = 0.f;
    {
      const uint16_t* po = a.o + b * a.sob + (int64_t)qi * a.sor + col;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int kk = 16 * s + 8 * h2;
        float x[8], y[8];
        unpack8<DT>(*reinterpret_cast<const uint4*>(po + (kk < a.d ? kk : 0)), x);
        unpack8<DT>(df[s], y);
        float p = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) p = fmaf(x[i], y[i], p);
        delta += kk < a.d ? p : 0.f;
      }
      delta += __shfl_xor(delta, 32, 64);
    }
    float l2 = a.lse_in[stat] * LOG2E;
    if (l2 == -INFINITY) l2 = INFINITY;  // a row without a key: P = exp2(0 - inf) = 0
    if (t < T && live && h2 == 0) a.delta[stat] = delta;
    f32x16 acc[OT];
#pragma unroll
    for (int i = 0; i < OT; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;

    auto tile = [&](int kr, bool masked) {
      f32x16 s, dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.f;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        s = HT<DT>::mfma32(*reinterpret_cast<const uint4*>(ks + (kr + li) * P + 16 * i + 8 * h2), qf[i], s);
        dp = HT<DT>::mfma32(*reinterpret_cast<const uint4*>(vs + (kr + li) * P + 16 * i + 8 * h2), df[i], dp);
      }
      if (masked) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const f32x4 m = *reinterpret_cast<const f32x4*>(bias + kr + 8 * c + 4 * h2);
#pragma unroll
          for (int r = 0; r < 4; ++r) s[4 * c + r] += m[r];
        }
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = fast_exp2(fmaf(s[r], a.c, -l2)) * (dp[r] - delta);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint4 ds = pack_k<DT>(s, u);
#pragma unroll
        for (int i = 0; i < OT; ++i) acc[i] = HT<DT>::mfma32(read_tr(ks, P, kr + 16 * u, 32 * i, lane), ds, acc[i]);
      }
    };
    if constexpr (RESIDENT) {
      for (int kr = 0; kr < len; kr += 32) tile(kr, a.mask || kr + 32 > len);
    } else {
      for (int k0 = 0; k0 < len; k0 += CH) {
        __syncthreads();
        stage_kv<KS, THREADS>(a, e, g, len, k0, CH, ks, vs, bias, tid);
        __syncthreads();
        if (t < T) {
          tile(0, a.mask || k0 + 32 > len);
          if (k0 + 32 < len) tile(32, a.mask || k0 + 64 > len);
        }
      }
    }
    if (t >= T) continue;
    uint16_t* p = a.out + b * a.sob + (int64_t)qi * a.sor + col;
#pragma unroll
    for (int i = 0; i < OT; ++i) store_tile<DT>(acc[i], a.scale, p, live, i, a.d, h2);
  }
}

// QT query rows per LDS buffer
constexpr int qt_rows(int ks) { return ks <= 5 ? 64 : 32; }
constexpr int dkv_lds(int ks) { return 2 * (2 * qt_rows(ks) * (16 * ks + 8) * 2 + 2 * qt_rows(ks) * 4 + 64); }

template <int DT, int KS, int NW>
__global__ __launch_bounds__(64 * NW, KS <= 5 ? 2 : 1) void xattn_dkv_kernel(const Args a) {
  constexpr int OT = (KS + 1) / 2, P = 16 * KS + 8, THREADS = 64 * NW, QT = qt_rows(KS), CHN = 2 * KS;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  constexpr int BUF = 2 * QT * P * 2 + 2 * QT * 4 + 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h2 = lane >> 5, li = lane & 31;
  // blocks of one XCD: the key heads of the same rows, then the key groups
  const unsigned L = xcd_remap(blockIdx.x, gridDim.x);
  const int g = (int)(L % (unsigned)a.kvh);
  const int kt = (int)(L / (unsigned)a.kvh) % a.nb, e = (int)(L / (unsigned)a.kvh) / a.nb;
  const int len = valid_len(a, e);
  const int key = (kt * NW + wave) * 32 + li;
  const bool valid = key_valid(a, e, len, min(key, a.Nk - 1)) && key < a.Nk;
  const bool any = (kt * NW + wave) * 32 < len;  // (wave-uniform)
  // flat rows of this part, in whole QT tiles
  const int T = (a.R + QT - 1) / QT, per = (T + a.nsplit - 1) / a.nsplit;
  const int t_lo = min(T, (int)blockIdx.y * per), t_hi = kt * NW * 32 < len ? min(T, t_lo + per) : t_lo;

  uint4 kf[KS], vf[KS];
  {
    const uint16_t* kp = a.k + (int64_t)e * a.skb + (int64_t)(valid ? key : 0) * a.skr + (int64_t)g * a.d;
    const uint16_t* vp = a.v + (int64_t)e * a.svb + (int64_t)(valid ? key : 0) * a.svr + (int64_t)g * a.d;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int kk = 16 * s + 8 * h2;
      kf[s] = vf[s] = make_uint4(0, 0, 0, 0);
      if (valid && kk < a.d) {
        kf[s] = *reinterpret_cast<const uint4*>(kp + kk);
        vf[s] = *reinterpret_cast<const uint4*>(vp + kk);
      }
    }
  }
  f32x16 dk[OT], dv[OT];
#pragma unroll
  for (int i = 0; i < OT; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) dk[i][r] = dv[i][r] = 0.f;

  // rows [QT t, QT t + QT) of q and dO, their lse (log2 units) and delta into buffer b; rows that do not exist: zeros, P = 0
  auto stage = [&](int t, int b) {
    uint16_t* qs = reinterpret_cast<uint16_t*>(smem + b * BUF);
    uint16_t* ds = qs + QT * P;
    float* l2 = reinterpret_cast<float*>(smem + b * BUF + 2 * QT * P * 2 + 64);
    for (int i = tid; i < QT * CHN; i += THREADS) {
      const int row = i / CHN, cc = (i - row * CHN) * 8, f = t * QT + row;
      uint4 x = make_uint4(0, 0, 0, 0), y = make_uint4(0, 0, 0, 0);
      if (f < a.R && cc < a.d) {
        int img, qi, hh;
        flat_row(a, f, img, qi, hh);
        const int64_t bb = (int64_t)e * a.G + img, col = (int64_t)(g * a.hg + hh) * a.d + cc;
        x = *reinterpret_cast<const uint4*>(a.q + bb * a.sqb + (int64_t)qi * a.sqr + col);
        y = *reinterpret_cast<const uint4*>(a.dout + bb * a.sdb + (int64_t)qi * a.sdr + col);
      }
      *reinterpret_cast<uint4*>(qs + row * P + cc) = x;
      *reinterpret_cast<uint4*>(ds + row * P + cc) = y;
    }
    for (int i = tid; i < QT; i += THREADS) {
      const int f = t * QT + i;
      float l = INFINITY, dl = 0.f;
      if (f < a.R) {
        int img, qi, hh;
        flat_row(a, f, img, qi, hh);
        const int64_t stat = (((int64_t)e * a.G + img) * a.kvh * a.hg + g * a.hg + hh) * a.Nq + qi;
        l = a.lse_in[stat] * LOG2E;
        l = l == -INFINITY ? INFINITY : l;
        dl = a.delta[stat];
      }
      l2[i] = l;
      l2[QT + i] = dl;
    }
  };
  if (t_lo < t_hi) stage(t_lo, 0);
  for (int t = t_lo; t < t_hi; ++t) {
    const int b = (t - t_lo) & 1;
    __syncthreads();
    if (t + 1 < t_hi) stage(t + 1, b ^ 1);
    if (!any) continue;
    const uint16_t* qs = reinterpret_cast<const uint16_t*>(smem + b * BUF);
    const uint16_t* ds = qs + QT * P;
    const float* l2 = reinterpret_cast<const float*>(smem + b * BUF + 2 * QT * P * 2 + 64);
#pragma unroll
    for (int q0 = 0; q0 < QT; q0 += 32) {
      f32x16 s, dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.f;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        s = HT<DT>::mfma32(*reinterpret_cast<const uint4*>(qs + (q0 + li) * P + 16 * i + 8 * h2), kf[i], s);
        dp = HT<DT>::mfma32(*reinterpret_cast<const uint4*>(ds + (q0 + li) * P + 16 * i + 8 * h2), vf[i], dp);
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const f32x4 l = *reinterpret_cast<const f32x4*>(l2 + q0 + 8 * c + 4 * h2);
        const f32x4 dl = *reinterpret_cast<const f32x4*>(l2 + QT + q0 + 8 * c + 4 * h2);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = fast_exp2(fmaf(s[4 * c + r], a.c, -l[r]));
          s[4 * c + r] = p;
          dp[4 * c + r] = p * (dp[4 * c + r] - dl[r]);
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint4 pf = pack_k<DT>(s, u), sf = pack_k<DT>(dp, u);
#pragma unroll
        for (int i = 0; i < OT; ++i) {
          dv[i] = HT<DT>::mfma32(read_tr(ds, P, q0 + 16 * u, 32 * i, lane), pf, dv[i]);
          dk[i] = HT<DT>::mfma32(read_tr(qs, P, q0 + 16 * u, 32 * i, lane), sf, dk[i]);
        }
      }
    }
  }
  if (key >= a.Nk) return;
  const int64_t C = (int64_t)a.kvh * a.d, at = ((int64_t)e * a.Nk + key) * C + (int64_t)g * a.d, plane = (int64_t)a.Be * a.Nk * C;
#pragma unroll
  for (int i = 0; i < OT; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int d0 = 32 * i + 8 * c + 4 * h2;
      if (d0 >= a.d) continue;
      f32x4 x, y;  // a key that the mask drops has no gradient (its columns hold what zeros gave)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[r] = valid ? dk[i][4 * c + r] * a.scale : 0.f;
        y[r] = valid ? dv[i][4 * c + r] : 0.f;
      }
      if (a.nsplit > 1) {
        float* w = a.ws + (int64_t)blockIdx.y * 2 * plane + at + d0;
        *reinterpret_cast<f32x4*>(w) = x;
        *reinterpret_cast<f32x4*>(w + plane) = y;
      } else {
        *reinterpret_cast<uint2*>(a.dk + at + d0) = make_uint2(pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3]));
        *reinterpret_cast<uint2*>(a.dv + at + d0) = make_uint2(pack2<DT>(y[0], y[1]), pack2<DT>(y[2], y[3]));
      }
    }
}

// dk / dv = the sum of the parts, in order
template <int DT>
__global__ __launch_bounds__(256) void xattn_dkv_join_kernel(const float* ws, uint16_t* dk, uint16_t* dv, int64_t plane, int parts) {
  const int64_t n4 = plane >> 2;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < 2 * n4; i += (int64_t)gridDim.x * 256) {
    const int64_t at = i < n4 ? i : i - n4;
    const float* w = ws + (i < n4 ? 0 : plane) + 4 * at;
    f32x4 s = *reinterpret_cast<const f32x4*>(w);
    for (int p = 1; p < parts; ++p) s += *reinterpret_cast<const f32x4*>(w + (int64_t)p * 2 * plane);
    *reinterpret_cast<uint2*>((i < n4 ? dk : dv) + 4 * at) = make_uint2(pack2<DT>(s[0], s[1]), pack2<DT>(s[2], s[3]));
  }
}

struct Plan {
  bool resident;
  int lds, nb;             // dq
  int nw, groups, nsplit;  // dk / dv
};
// dq: as the forward.  dk / dv: as many waves per block as there are key tiles (1, 2 or 4), the rows cut into parts until two
// blocks per CU have work and a part keeps at least four tiles.
Plan plan(const Args& a) {
  Plan p{};
  const int ks = k_steps(a.d), cus = cu_count(), eg = a.Be * a.kvh;
  const int npad = (a.Nk + 31) / 32 * 32;
  p.resident = kv_lds(ks, npad) <= RES_LDS;
  p.lds = p.resident ? kv_lds(ks, npad) : kv_lds(ks, CH);
  const int most = ((a.R + 31) / 32 + 3) / 4, want = p.resident ? 4 * cus : most * eg;
  p.nb = (want + eg - 1) / eg;
  if (p.nb > most) p.nb = most;
  const int tiles = a.Nk > 0 ? (a.Nk + 31) / 32 : 1;  // (without keys there is no dk / dv launch)
  p.nw = tiles <= 1 ? 1 : tiles == 2 ? 2 : 4;
  p.groups = (tiles + p.nw - 1) / p.nw;
  const int T = (a.R + qt_rows(ks) - 1) / qt_rows(ks);
  const int64_t blocks = (int64_t)eg * p.groups;
  int64_t n = ((int64_t)(p.nw == 4 ? 2 : p.nw == 2 ? 4 : 8) * cus + blocks - 1) / blocks;
  if (n > T / 4) n = T / 4;
  if (n > 256) n = 256;
  p.nsplit = n < 1 ? 1 : (int)n;
  return p;
}

// workspace: delta [B, heads, Nq], then the parts' dk / dv
int64_t delta_floats(const Args& a) { return ((int64_t)a.Be * a.kvh * a.R + 3) / 4 * 4; }
size_t ws_bytes(const Args& a, const Plan& p) {
  const int64_t parts = p.nsplit > 1 ? (int64_t)p.nsplit * 2 * a.Be * a.Nk * a.kvh * a.d : 0;
  return (size_t)(delta_floats(a) + parts) * sizeof(float);
}

template <int DT, int KS>
int launch(Args& a, const Plan& p, hipStream_t st) {
  const unsigned eg = (unsigned)(a.Be * a.kvh);
  a.nb = p.nb; a.nsplit = 1;
  if (p.resident) hipLaunchKernelGGL((xattn_dq_kernel<DT, KS, true>), dim3(eg * (unsigned)p.nb), dim3(256), p.lds, st, a);
  else hipLaunchKernelGGL((xattn_dq_kernel<DT, KS, false>), dim3(eg * (unsigned)p.nb), dim3(256), p.lds, st, a);
  MIMO_LAUNCH_CHECK();
  if (a.Nk == 0) return MIMO_OK;
  a.nb = p.groups; a.nsplit = p.nsplit;
  const dim3 grid(eg * (unsigned)p.groups, (unsigned)p.nsplit);
  constexpr int lds = dkv_lds(KS);
  if (p.nw == 1) hipLaunchKernelGGL((xattn_dkv_kernel<DT, KS, 1>), grid, dim3(64), lds, st, a);
  else if (p.nw == 2) hipLaunchKernelGGL((xattn_dkv_kernel<DT, KS, 2>), grid, dim3(128), lds, st, a);
  else hipLaunchKernelGGL((xattn_dkv_kernel<DT, KS, 4>), grid, dim3(256), lds, st, a);
  MIMO_LAUNCH_CHECK();
  if (p.nsplit > 1) {
    const int64_t plane = (int64_t)a.Be * a.Nk * a.kvh * a.d, nwg = (plane / 2 + 255) / 256;
    hipLaunchKernelGGL((xattn_dkv_join_kernel<DT>), dim3((unsigned)(nwg > 2048 ? 2048 : nwg)), dim3(256), 0, st, a.ws, a.dk, a.dv, plane,
                       p.nsplit);
    MIMO_LAUNCH_CHECK();
  }
  return MIMO_OK;
}

template <int DT>
int dispatch(Args& a, const Plan& p, hipStream_t st) {
  int rc = MIMO_EINVAL;
#define CALL(KS) rc = launch<DT, KS>(a, p, st)
  MIMO_XATTN_DISPATCH(k_steps(a.d), CALL)
#undef CALL
  return rc;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace mimo_xattn

extern "C" size_t mimo_cross_attention_backward_workspace(const mimo_cross_attention_params* p) {
  mimo_xattn::Args a{};
  if (mimo_xattn::fill(a, p) != MIMO_OK) return 0;
  return mimo_xattn::ws_bytes(a, mimo_xattn::plan(a));
}

extern "C" int mimo_cross_attention_backward(int dtype, const void* dout, const void* q, const void* k, const void* v, const void* out,
                                             const float* lse, void* dq, void* dk, void* dv, const mimo_cross_attention_params* p,
                                             void* workspace, size_t workspace_bytes, void* stream) {
  using namespace mimo_xattn;
  Args a{};
  if (const int rc = fill(a, p)) return rc;
  if ((a.sdb & 7) || (a.sdr & 7)) return MIMO_EINVAL;
  if (!dout || !q || !out || !lse || !dq || !workspace || (a.Nk > 0 && (!k || !v || !dk || !dv))) return MIMO_EINVAL;
  if (!aligned16(dout) || !aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(dq) || !aligned16(dk) ||
      !aligned16(dv) || !aligned16(workspace))
    return MIMO_EINVAL;
  a.dout = (const uint16_t*)dout; a.q = (const uint16_t*)q; a.k = (const uint16_t*)k; a.v = (const uint16_t*)v;
  a.o = (const uint16_t*)out; a.lse_in = lse; a.out = (uint16_t*)dq; a.dk = (uint16_t*)dk; a.dv = (uint16_t*)dv;
  const Plan pl = plan(a);
  if (workspace_bytes < ws_bytes(a, pl)) return MIMO_EINVAL;
  a.delta = (float*)workspace;
  a.ws = (float*)workspace + delta_floats(a);
  if (dtype == MIMO_F16) return dispatch<MIMO_F16>(a, pl, (hipStream_t)stream);
  if (dtype == MIMO_BF16) return dispatch<MIMO_BF16>(a, pl, (hipStream_t)stream);
  return MIMO_EDTYPE;
}
