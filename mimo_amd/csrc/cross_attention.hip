// cross_attention.hip — attention of a batch of images to an encoder's states of another length (gfx950, MFMA 32x32x16).
//
//   out[q] = sum_k softmax_k(scale q.k + mask) v[k],  lse[q] = ln sum_k exp(scale q.k + mask);  a row without a key gives 0, -inf
//
// One pass with a running maximum and sum per query (fp32); the products are S^T = K.Q^T and O^T = V^T.P^T, so a lane owns one
// query and the packed scores are the second product's operand as they stand.  P is rounded to the operand type for that
// product (one rounding of the size of the output's own), the sum is taken in fp32 before it.
//
// What bounds it: 4 Nk flops per byte of q and out.  Up to some 200 keys the call is a stream of q and out through the chip, so
// the keys of a (row, head) are staged in LDS ONCE per block and the block walks many query tiles over them
// (xattn_kernel<RESIDENT>): no barrier after the first, the next tile's queries requested before this one's products.
// Longer key sequences stream through two LDS buffers of 64 keys that four query tiles share (RESIDENT = false), and when the
// query tiles are too few to fill the chip the keys are cut into parts (gridDim.y) joined by xattn_join_kernel in a fixed order.
#include "cross_attention.hip.h"

namespace mimo_xattn {

int fill(Args& a, const mimo_cross_attention_params* p) {
  if (!p || p->B <= 0 || p->Be <= 0 || p->B % p->Be || p->Nq <= 0 || p->Nk < 0 || p->heads <= 0 || p->kv_heads <= 0 ||
      p->heads % p->kv_heads || p->d <= 0 || p->d > 160 || (p->d & 7) || !(p->scale > 0.f))
    return MIMO_EINVAL;
  if ((p->q_batch & 7) || (p->q_row & 7) || (p->k_batch & 7) || (p->k_row & 7) || (p->v_batch & 7) || (p->v_row & 7)) return MIMO_EINVAL;
  a.Be = p->Be; a.G = p->B / p->Be; a.Nq = p->Nq; a.Nk = p->Nk; a.kvh = p->kv_heads; a.hg = p->heads / p->kv_heads; a.d = p->d;
  const int64_t R = (int64_t)a.G * a.Nq * a.hg;
  if (R >= 0x40000000LL || (int64_t)p->Be * p->kv_heads >= 0x10000 || p->Nk >= 0x40000000) return MIMO_EINVAL;
  a.R = (int)R;
  a.by_hg = fast_div((uint32_t)a.hg); a.by_nq = fast_div((uint32_t)a.Nq);
  a.scale = p->scale; a.c = p->scale * LOG2E;
  a.sqb = p->q_batch; a.sqr = p->q_row; a.skb = p->k_batch; a.skr = p->k_row; a.svb = p->v_batch; a.svr = p->v_row;
  a.smb = p->mask_row;
  const int64_t C = (int64_t)p->heads * p->d;
  a.sor = C; a.sob = C * p->Nq;
  a.sdr = p->dout_row; a.sdb = p->dout_batch;
  a.kv_len = p->kv_len; a.mask = (const uint8_t*)p->mask;
  return MIMO_OK;
}

namespace {

template <int V>
struct IC {
  static constexpr int value = V;
};

constexpr int CH = 64;          // keys per streamed buffer
constexpr int RES_LDS = 80000;  // resident keys: two blocks per CU

inline int lds_of(int ks, bool resident, int nk) { return resident ? kv_lds(ks, (nk + 31) / 32 * 32) : 2 * kv_lds(ks, CH); }

template <int DT, int KS, bool RESIDENT, int NW>
__global__ __launch_bounds__(64 * NW, KS <= 4 ? 3 : 2) void xattn_kernel(const Args a) {
  constexpr int OT = (KS + 1) / 2, P = 16 * KS + 8, THREADS = 64 * NW;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h2 = lane >> 5, li = lane & 31;
  // consecutive blocks of an XCD are the key heads of the same query rows: they read the same lines of q
  const unsigned L = xcd_remap(blockIdx.x, gridDim.x);
  const int g = (int)(L % (unsigned)a.kvh);
  const int j = (int)(L / (unsigned)a.kvh) % a.nb, e = (int)(L / (unsigned)a.kvh) / a.nb;
  const int len = valid_len(a, e);
  const int T = (a.R + 31) >> 5;  // query tiles of this (e, g)
  // keys of this part
  const int per = ((len + CH - 1) / CH + a.nsplit - 1) / a.nsplit * CH;
  const int k_lo = min(len, (int)blockIdx.y * per), k_hi = min(len, k_lo + per);
  const int nkeys = k_hi - k_lo;

  const int npad = RESIDENT ? (a.Nk + 31) / 32 * 32 : CH;
  uint16_t* const ks0 = reinterpret_cast<uint16_t*>(smem);
  uint16_t* const vs0 = ks0 + npad * P;
  float* const bias0 = reinterpret_cast<float*>(smem + 2 * npad * P * 2 + 64);
  const int stride = kv_lds(KS, npad);  // bytes between the two streamed buffers

  if constexpr (RESIDENT) {
    stage_kv<KS, THREADS>(a, e, g, len, 0, (len + 31) / 32 * 32, ks0, vs0, bias0, tid);
    __syncthreads();
  }
  // a streamed block's waves share its key buffers: all of them walk the same number of tiles
  const int step = a.nb * NW;
  int t = j * NW + wave;
  const int rounds = RESIDENT ? 0 : (T - j * NW + step - 1) / step;

  uint4 qf[KS], qn[KS];
  auto query = [&](int tt, uint4 (&f)[KS]) {
    int img, qi, hh;
    flat_row(a, min(32 * tt + li, a.R - 1), img, qi, hh);
    load_row<KS>(f, a.q + ((int64_t)e * a.G + img) * a.sqb + (int64_t)qi * a.sqr + (int64_t)(g * a.hg + hh) * a.d, a.d, h2);
  };
  if (t < T) query(t, qn);

  for (int round = 0; RESIDENT ? t < T : round < rounds; t += step, ++round) {
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = qn[s];
    if (t + step < T) query(t + step, qn);
    f32x16 ot[OT];
#pragma unroll
    for (int i = 0; i < OT; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) ot[i][r] = 0.f;
    float m_run = -INFINITY, l_run = 0.f;

    // two 32-key tiles at LDS rows kr.. (n = how many of them hold keys)
    auto tiles = [&](const uint16_t* ks, const uint16_t* vs, const float* bias, int kr, auto n_c, bool masked) {
      constexpr int n = decltype(n_c)::value;
      f32x16 st[n];
#pragma unroll
      for (int u = 0; u < n; ++u) {
#pragma unroll
        for (int r = 0; r < 16; ++r) st[u][r] = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s)
          st[u] = HT<DT>::mfma32(*reinterpret_cast<const uint4*>(ks + (kr + 32 * u + li) * P + 16 * s + 8 * h2), qf[s], st[u]);
      }
      if (masked) {
#pragma unroll
        for (int u = 0; u < n; ++u)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const f32x4 b = *reinterpret_cast<const f32x4*>(bias + kr + 32 * u + 8 * c + 4 * h2);
#pragma unroll
            for (int r = 0; r < 4; ++r) st[u][4 * c + r] += b[r];
          }
      }
      float mt = st[0][0];
#pragma unroll
      for (int u = 0; u < n; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) mt = fmaxf(mt, st[u][r]);
      mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
      const float m_new = fmaxf(m_run, mt);
      const float m_use = m_new == -INFINITY ? 0.f : m_new;  // nothing but masked keys so far: exp2(-inf) below
      if (__builtin_amdgcn_ballot_w64(m_new > m_run) != 0ull) {
        const float alpha = fast_exp2((m_run - m_use) * a.c);
        l_run *= alpha;
#pragma unroll
        for (int i = 0; i < OT; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) ot[i][r] *= alpha;
      }
      m_run = m_new;
      const float mc = -m_use * a.c;
      float ps = 0.f;
#pragma unroll
      for (int u = 0; u < n; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          st[u][r] = fast_exp2(fmaf(st[u][r], a.c, mc));
          ps += st[u][r];
        }
      l_run += ps;  // this lane's half of the keys; the halves meet at the end
#pragma unroll
      for (int u = 0; u < 2 * n; ++u) {
        const uint4 pf = pack_k<DT>(st[u >> 1], u & 1);
#pragma unroll
        for (int i = 0; i < OT; ++i) ot[i] = HT<DT>::mfma32(read_tr(vs, P, kr + 16 * u, 32 * i, lane), pf, ot[i]);
      }
    };
    if constexpr (RESIDENT) {
      int kr = 0;
      for (; kr + 32 < len; kr += 64) tiles(ks0, vs0, bias0, kr, IC<2>{}, a.mask || kr + 64 > len);
      if (kr < len) tiles(ks0, vs0, bias0, kr, IC<1>{}, a.mask || kr + 32 > len);
    } else {
      // buffer b holds chunk i (i & 1 == b); the other one is filled while this one is used, one barrier per chunk
      const int chunks = (nkeys + CH - 1) / CH;
      __syncthreads();  // the previous round's last chunk is read
      if (chunks > 0) stage_kv<KS, THREADS>(a, e, g, k_hi, k_lo, CH, ks0, vs0, bias0, tid);
      for (int i = 0; i < chunks; ++i) {
        __syncthreads();
        const int off = (i & 1) * stride, nxt = ((i + 1) & 1) * stride;
        auto at = [&](const void* p, int o) { return (unsigned char*)p + o; };
        if (i + 1 < chunks)
          stage_kv<KS, THREADS>(a, e, g, k_hi, k_lo + (i + 1) * CH, CH, (uint16_t*)at(ks0, nxt), (uint16_t*)at(vs0, nxt),
                                (float*)at(bias0, nxt), tid);
        if (t < T)
          tiles((const uint16_t*)at(ks0, off), (const uint16_t*)at(vs0, off), (const float*)at(bias0, off), 0, IC<2>{},
                a.mask || (i + 1) * CH > nkeys);
      }
    }
    if (t >= T) continue;
    l_run += __shfl_xor(l_run, 32, 64);
    const int f = 32 * t + li;
    const bool live = f < a.R;
    int img, qi, hh;
    flat_row(a, min(f, a.R - 1), img, qi, hh);
    const int head = g * a.hg + hh;
    const int64_t b = (int64_t)e * a.G + img;
    if (a.nsplit > 1) {  // partial: unnormalised rows, then (reference maximum in log2 units, sum)
      const int64_t row = (((int64_t)blockIdx.y * a.Be + e) * a.kvh + g) * a.R + f;
      float* po = a.ws + row * a.d;
      if (live) {
#pragma unroll
        for (int i = 0; i < OT; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int d0 = 32 * i + 8 * c + 4 * h2;
            if (d0 < a.d) *reinterpret_cast<f32x4*>(po + d0) = (f32x4){ot[i][4 * c], ot[i][4 * c + 1], ot[i][4 * c + 2], ot[i][4 * c + 3]};
          }
        if (h2 == 0) {
          float* ml = a.ws + (int64_t)a.nsplit * a.Be * a.kvh * a.R * a.d + 2 * row;
          ml[0] = m_run * a.c;
          ml[1] = l_run;
        }
      }
      continue;
    }
    const float inv = l_run > 0.f ? 1.f / l_run : 0.f;
    uint16_t* p = a.out + b * a.sob + (int64_t)qi * a.sor + (int64_t)head * a.d;
#pragma unroll
    for (int i = 0; i < OT; ++i) store_tile<DT>(ot[i], inv, p, live, i, a.d, h2);
    if (a.lse && live && h2 == 0)
      a.lse[(b * a.kvh * a.hg + head) * a.Nq + qi] = l_run > 0.f ? m_run * a.scale + logf(l_run) : -INFINITY;
  }
}

// joins the parts of the keys: out = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s, parts in order.  One thread per row and four
// channels.
template <int DT>
__global__ __launch_bounds__(256) void xattn_join_kernel(const Args a) {
  const int d4 = a.d >> 2;
  const int64_t rows = (int64_t)a.Be * a.kvh * a.R, total = rows * d4;
  const float* mls = a.ws + (int64_t)a.nsplit * rows * a.d;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / d4;
    const int c = (int)(i - row * d4) * 4;
    float m = -INFINITY;
    for (int s = 0; s < a.nsplit; ++s) m = fmaxf(m, mls[2 * ((int64_t)s * rows + row)]);
    const float mu = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < a.nsplit; ++s) {
      const float* ml = mls + 2 * ((int64_t)s * rows + row);
      const float w = fast_exp2(ml[0] - mu);
      l = fmaf(w, ml[1], l);
      o += *reinterpret_cast<const f32x4*>(a.ws + ((int64_t)s * rows + row) * a.d + c) * w;
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    const int64_t eg = row / a.R;
    const int g = (int)(eg % a.kvh);
    int img, qi, hh;
    flat_row(a, (int)(row - eg * a.R), img, qi, hh);
    const int64_t b = eg / a.kvh * a.G + img;
    const int head = g * a.hg + hh;
    *reinterpret_cast<uint2*>(a.out + b * a.sob + (int64_t)qi * a.sor + (int64_t)head * a.d + c) =
        make_uint2(pack2<DT>(o[0] * inv, o[1] * inv), pack2<DT>(o[2] * inv, o[3] * inv));
    if (a.lse && c == 0) a.lse[(b * a.kvh * a.hg + head) * a.Nq + qi] = l > 0.f ? (mu + log2f(l)) * LN2 : -INFINITY;
  }
}

struct Plan {
  bool resident;
  int nw, nb, nsplit, lds;
};
// Resident keys while two blocks of them fit a CU.  Blocks: enough for three rounds of every CU at the LDS each takes, never
// more than one per NW query tiles.  Streamed with one wave per block when one tile holds all queries (the other waves would
// only wait), else four; the keys are cut while the blocks do not fill the chip and a part keeps at least 256 keys.
Plan plan(const Args& a) {
  Plan p{};
  const int ks = k_steps(a.d), cus = cu_count();
  const int T = (a.R + 31) / 32;
  p.resident = lds_of(ks, true, a.Nk) <= RES_LDS;
  p.nw = (!p.resident && T == 1) ? 1 : 4;
  p.lds = lds_of(ks, p.resident, a.Nk);
  const int most = (T + p.nw - 1) / p.nw, eg = a.Be * a.kvh;
  if (p.resident) {
    const int want = 4 * cus;
    p.nb = (want + eg - 1) / eg;
    if (p.nb > most) p.nb = most;
    p.nsplit = 1;
  } else {
    p.nb = most;
    const int64_t blocks = (int64_t)eg * most, fill = p.nw == 1 ? 8 * cus : 2 * cus;
    int64_t n = (fill + blocks - 1) / blocks;
    const int parts = (a.Nk + 255) / 256;
    if (n > parts) n = parts;
    if (n > 64) n = 64;
    p.nsplit = n < 1 ? 1 : (int)n;
  }
  return p;
}

size_t ws_bytes(const Args& a, const Plan& p) {
  return p.nsplit > 1 ? (size_t)p.nsplit * a.Be * a.kvh * a.R * (a.d + 2) * sizeof(float) : 0;
}

template <int DT, int KS>
int launch(const Args& a, const Plan& p, hipStream_t st) {
  const dim3 grid((unsigned)(a.Be * a.kvh) * (unsigned)p.nb, (unsigned)p.nsplit);
  if (p.resident) hipLaunchKernelGGL((xattn_kernel<DT, KS, true, 4>), grid, dim3(256), p.lds, st, a);
  else if (p.nw == 1) hipLaunchKernelGGL((xattn_kernel<DT, KS, false, 1>), grid, dim3(64), p.lds, st, a);
  else hipLaunchKernelGGL((xattn_kernel<DT, KS, false, 4>), grid, dim3(256), p.lds, st, a);
  MIMO_LAUNCH_CHECK();
  if (p.nsplit > 1) {
    const int64_t total = (int64_t)a.Be * a.kvh * a.R * (a.d / 4), nwg = (total + 255) / 256;
    hipLaunchKernelGGL((xattn_join_kernel<DT>), dim3((unsigned)(nwg > 4096 ? 4096 : nwg)), dim3(256), 0, st, a);
    MIMO_LAUNCH_CHECK();
  }
  return MIMO_OK;
}

template <int DT>
int dispatch(const Args& a, const Plan& p, hipStream_t st) {
  int rc = MIMO_EINVAL;
#define CALL(KS) rc = launch<DT, KS>(a, p, st)
  MIMO_XATTN_DISPATCH(k_steps(a.d), CALL)
#undef CALL
  return rc;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace mimo_xattn

extern "C" size_t mimo_cross_attention_workspace(const mimo_cross_attention_params* p) {
  mimo_xattn::Args a{};
  if (mimo_xattn::fill(a, p) != MIMO_OK) return 0;
  return mimo_xattn::ws_bytes(a, mimo_xattn::plan(a));
}

extern "C" int mimo_cross_attention(int dtype, const void* q, const void* k, const void* v, void* out, float* lse,
                                    const mimo_cross_attention_params* p, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace mimo_xattn;
  Args a{};
  if (const int rc = fill(a, p)) return rc;
  if (!q || !out || (a.Nk > 0 && (!k || !v)) || !aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out)) return MIMO_EINVAL;
  a.q = (const uint16_t*)q; a.k = (const uint16_t*)k; a.v = (const uint16_t*)v; a.out = (uint16_t*)out; a.lse = lse;
  const Plan pl = plan(a);
  a.nb = pl.nb; a.nsplit = pl.nsplit;
  if (ws_bytes(a, pl) > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < ws_bytes(a, pl))) return MIMO_EINVAL;
  a.ws = (float*)workspace;
  if (dtype == MIMO_F16) return dispatch<MIMO_F16>(a, pl, (hipStream_t)stream);
  if (dtype == MIMO_BF16) return dispatch<MIMO_BF16>(a, pl, (hipStream_t)stream);
  return MIMO_EDTYPE;
}
