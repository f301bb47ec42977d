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
// Measured: 48 x 4096 queries, 8 heads of 40, 77 keys in 95 us (2.6 TB/s).  Neither the products (14 % of it) nor the vector
// instructions (50 %) bound that but the 80-byte piece that a head has of a row: a copy of such pieces, a row per lane, takes 90 to
// 103 us, of 320-byte pieces 53, of whole rows 36 to 41.  48 x 1024 queries, 8 heads of 80, 257 keys in 54 us, 60 with a mask: products
// and exponentials in turn.
// Longer key sequences stream through two LDS buffers of 64 keys that four query tiles share (RESIDENT = false), and when the
// query tiles are too few to fill the chip the keys are cut into parts (gridDim.y) joined by xattn_join_kernel in a fixed order.
#include "cross_attention.hip.h"

namespace mimo_xattn {

int fill(Args& a, const mimo_cross_attention_params* p) {
  if (!p || p->B <= 0 || p->Be <= 0 || p->B % p->Be || p->Nq <= 0 || p->Nk < 0 || p->heads <= 0 || p->kv_heads <= 0 ||
      p->heads % p->kv_heads || p->d <= 0 || p->d > 160 || (p->d & 7) || !(p->scale >= 0x1p-126f && p->scale <= 0x1p126f))
    return MIMO_EINVAL;
  if ((p->q_batch & 7) || (p->q_row & 7) || (p->k_batch & 7) || (p->k_row & 7) || (p->v_batch & 7) || (p->v_row & 7)) return MIMO_EINVAL;
  a.Be = p->Be; a.G = p->B / p->Be; a.Nq = p->Nq; a.Nk = p->Nk; a.kvh = p->kv_heads; a.hg = p->heads / p->kv_heads; a.d = p->d;
  const int64_t R = (int64_t)a.G * a.Nq * a.hg;
  if (R >= 0x40000000LL || (int64_t)p->Be * p->kv_heads >= 0x10000 || p->Nk >= 0x40000000 || (int64_t)p->heads * p->Nq >= 0x8000000 ||
      p->heads >= 0x10000)
    return MIMO_EINVAL;
  a.R = (int)R;
  a.by_hg = fast_div((uint32_t)a.hg); a.by_nq = fast_div((uint32_t)a.Nq); a.by_dc = fast_div((uint32_t)a.d / 8);
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

// keys per streamed buffer: what a thread can hold on its way
constexpr int stream_keys(int ks, int nw) { return ks >= 8 || (nw == 1 && ks > 4) ? 32 : 64; }

constexpr float LAG = 8.f;  // log2 units by which a row's maximum may pass its reference before the row is rescaled (48 x 1024 queries, 8 heads of 80, 257 keys: 54.2 us, with 0 56.4)

// RESIDENT: all keys of (e, g) staged once; NW = 4 (two or more blocks per CU) or 8 (one).  Else: streamed in chunks of CHK keys
// through two buffers, NW = 4 or 1 waves that share them.
template <int DT, int KS, bool RESIDENT, int NW, int CHK>
__global__ __launch_bounds__(64 * NW, NW == 8 ? 2 : NW == 1 && KS >= 8 ? 1 : (KS <= 3 && NW > 1) || KS == 2 || (KS == 4 && RESIDENT) ? 3 : 2) void xattn_kernel(const Args a) {
  constexpr int OT = (KS + 1) / 2, P = 16 * KS + 8, THREADS = 64 * NW;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h2 = lane >> 5, li = lane & 31;
  // consecutive blocks of an XCD are the key heads of the same query rows: they share the lines of q and out; then come the encoder
  // rows, whose lengths differ: every XCD gets some of each
  const unsigned L = xcd_remap(blockIdx.x, gridDim.x);
  const int g = (int)(L % (unsigned)a.kvh);
  const int e = (int)(L / (unsigned)a.kvh) % a.Be, j = (int)(L / (unsigned)a.kvh) / a.Be;
  const int len = valid_len(a, e);
  const int T = (a.R + 31) >> 5;  // query tiles of this (e, g)
  // keys of this part
  const int per = ((len + CHK - 1) / CHK + a.nsplit - 1) / a.nsplit * CHK;
  const int k_lo = min(len, (int)blockIdx.y * per), k_hi = min(len, k_lo + per);
  const bool ones = (a.d & 31) != 0;  // the last channel tile has a row to spare: the sum of P comes with the product

  const int npad = RESIDENT ? (a.Nk + 31) / 32 * 32 : CHK;
  const int stride = kv_lds(KS, npad);  // bytes between the two streamed buffers
  auto ks_of = [&](int b) { return reinterpret_cast<uint16_t*>(smem + b * stride); };
  auto vs_of = [&](int b) { return reinterpret_cast<uint16_t*>(smem + b * stride) + npad * P; };
  auto bias_of = [&](int b) { return reinterpret_cast<float*>(smem + b * stride + 2 * npad * P * 2 + 64); };

  Stager<KS, THREADS, CHK> stager;
  stager.open(a, e, g);
  if constexpr (RESIDENT) {
    stage_all<DT, KS, THREADS>(a, e, g, len, ks_of(0), vs_of(0), bias_of(0), ones, tid);
    lds_barrier();
  }
  const int step = a.nb * NW;
  int t = j * NW + wave;

  uint4 qf[KS], qn[RESIDENT ? KS : 1];
  auto query = [&](int tt, auto& f) {
    int img, qi, hh;
    flat_row(a, min(32 * tt + li, a.R - 1), img, qi, hh);
    load_row<KS>(f, a.q + ((int64_t)e * a.G + img) * a.sqb + (int64_t)qi * a.sqr + (int64_t)(g * a.hg + hh) * a.d, a.d, h2);
  };
  if constexpr (RESIDENT) {
    if (t < T) query(t, qn);
  }

  // (a streamed block has one tile per wave; its waves share the key buffers, so one without a tile goes through the chunks as well)
  for (bool first = true; RESIDENT ? t < T : first; t += step, first = false) {
    if constexpr (RESIDENT) {
#pragma unroll
      for (int s = 0; s < KS; ++s) qf[s] = qn[s];
      if (t + step < T) query(t + step, qn);
    } else {
      query(min(t, T - 1), qf);
    }
    f32x16 ot[OT];
#pragma unroll
    for (int i = 0; i < OT; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) ot[i][r] = 0.f;
    // m_ref: the maximum that P is taken against.  It follows the running maximum only when that passes it by LAG (P then stays
    // below 2^LAG: the same arithmetic, far fewer rescalings); sum: this lane's half of the keys
    float m_ref = -INFINITY, sum = 0.f;

    // two or one 32-key tiles at LDS rows kr..
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
      const bool move = mt > m_ref + a.lag;  // (m_ref = -inf: any finite maximum)
      const float old = m_ref;
      m_ref = move ? mt : old;
      if (__builtin_amdgcn_ballot_w64(move && old != -INFINITY) != 0ull) {  // (nothing is summed yet against -inf)
        const float alpha = move && old != -INFINITY ? fast_exp2((old - mt) * a.c) : 1.f;
        sum *= alpha;
#pragma unroll
        for (int i = 0; i < OT; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) ot[i][r] *= alpha;
      }
      const float mc = m_ref == -INFINITY ? 0.f : -m_ref * a.c;  // nothing but masked keys so far: exp2(-inf)
#pragma unroll
      for (int u = 0; u < n; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) st[u][r] = fast_exp2(fmaf(st[u][r], a.c, mc));
      if (!ones || a.lse) {
        float ps = 0.f;
#pragma unroll
        for (int u = 0; u < n; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r) ps += st[u][r];
        sum += ps;
      }
#pragma unroll
      for (int u = 0; u < 2 * n; ++u) {
        const uint4 pf = pack_k<DT>(st[u >> 1], u & 1);
#pragma unroll
        for (int i = 0; i < OT; ++i) ot[i] = HT<DT>::mfma32(read_tr(vs, P, kr + 16 * u, 32 * i, lane), pf, ot[i]);
      }
    };
    if constexpr (RESIDENT) {
      int kr = 0;
      for (; kr + 32 < len; kr += 64) tiles(ks_of(0), vs_of(0), bias_of(0), kr, IC<2>{}, a.mask || kr + 64 > len);
      if (kr < len) tiles(ks_of(0), vs_of(0), bias_of(0), kr, IC<1>{}, a.mask || kr + 32 > len);
    } else {
      // chunk i is in buffer i & 1; while it is used the next one is on its way into registers and then into the other buffer:
      // one barrier per chunk
      const int chunks = (k_hi - k_lo + CHK - 1) / CHK;
      if (chunks > 0) {
        stager.issue(a, e, k_hi, k_lo, tid);
        stager.template commit<DT>(a, ks_of(0), vs_of(0), bias_of(0), ones, tid);
        settle<KS>(qf);
        if (chunks > 1) stager.issue(a, e, k_hi, k_lo + CHK, tid);
      }
      for (int i = 0; i < chunks; ++i) {
        lds_barrier();
        const int b = i & 1;
        if (t < T) tiles(ks_of(b), vs_of(b), bias_of(b), 0, IC<CHK / 32>{}, a.mask || k_lo + (i + 1) * CHK > k_hi);
        if (i + 1 < chunks) {
          stager.template commit<DT>(a, ks_of(b ^ 1), vs_of(b ^ 1), bias_of(b ^ 1), ones, tid);
          if (i + 2 < chunks) stager.issue(a, e, k_hi, k_lo + (i + 2) * CHK, tid);
        }
      }
    }
    if (t >= T) continue;
    sum += __shfl_xor(sum, 32, 64);
    float l = sum;  // what the output is divided by: the sum of the P that were multiplied, where it came with them
    if (ones) {
      const int r = (a.d & 31) >> 3;  // row d of O^T: register 4 r of the last tile, lanes 0..31
      l = __shfl(r == 1 ? ot[OT - 1][4] : r == 2 ? ot[OT - 1][8] : ot[OT - 1][12], li, 64);
    }
    if constexpr (!RESIDENT) {
      if (a.nsplit > 1) {  // partial: unnormalised rows, then (reference maximum in log2 units, divisor, sum)
        const int f = 32 * t + li;
        const int64_t row = (((int64_t)blockIdx.y * a.Be + e) * a.kvh + g) * a.R + f;
        float* po = a.ws + row * a.d;
        if (f < a.R) {
#pragma unroll
          for (int i = 0; i < OT; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int d0 = 32 * i + 8 * c + 4 * h2;
              if (d0 < a.d)
                *reinterpret_cast<f32x4*>(po + d0) = (f32x4){ot[i][4 * c], ot[i][4 * c + 1], ot[i][4 * c + 2], ot[i][4 * c + 3]};
            }
          if (h2 == 0)
            *reinterpret_cast<f32x4*>(a.ws + (int64_t)a.nsplit * a.Be * a.kvh * a.R * a.d + 4 * row) = (f32x4){m_ref * a.c, l, sum, 0.f};
        }
        continue;
      }
    }
    const RowPlace place = row_place(a, e, g, t, li, a.out, a.lse);
    const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int i = 0; i < OT; ++i) store_tile<DT>(ot[i], inv, place, i, a.d, h2);
    if (a.lse) {
      const float v = sum > 0.f ? m_ref * a.scale + logf(sum) : -INFINITY;
      __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, v), place.table, h2 == 0 ? place.stat : 0xF0000000u, 0, 0);
    }
  }
}

// joins the parts of the keys: out = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s, parts in order.  A block takes 1024 / d rows
// (d / 4 threads each), the parts' (m, l, sum) pass through LDS once.
template <int DT>
__global__ __launch_bounds__(256) void xattn_join_kernel(const Args a) {
  __shared__ f32x4 part[32 * 64];  // [rows of the block][parts]
  const int d4 = a.d >> 2, per = 256 / d4 < 32 ? 256 / d4 : 32, n = a.nsplit;
  const int64_t rows = (int64_t)a.Be * a.kvh * a.R, row0 = (int64_t)blockIdx.x * per;
  const f32x4* mls = reinterpret_cast<const f32x4*>(a.ws + (int64_t)n * rows * a.d);
  for (int i = threadIdx.x; i < per * n; i += 256) {
    const int s = i / per, r = i - s * per;
    if (row0 + r < rows) part[r * n + s] = mls[(int64_t)s * rows + row0 + r];
  }
  const int r = threadIdx.x / d4, c = (threadIdx.x - r * d4) * 4;
  const int64_t row = row0 + r;
  const bool mine = r < per && row < rows;
  f32x4 x[8];
  const float* src = a.ws + row * a.d + c;
  if (mine) {
#pragma unroll
    for (int s = 0; s < 8; ++s)
      if (s < n) x[s] = *reinterpret_cast<const f32x4*>(src + (int64_t)s * rows * a.d);
  }
  lds_barrier();
  if (!mine) return;
  float m = -INFINITY;
  for (int s = 0; s < n; ++s) m = fmaxf(m, part[r * n + s][0]);
  const float mu = m == -INFINITY ? 0.f : m;
  float l = 0.f, sum = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < n; s0 += 8) {
#pragma unroll
    for (int s = 0; s < 8; ++s)
      if (s0 + s < n) {
        const f32x4 q = part[r * n + s0 + s];
        const float w = fast_exp2(q[0] - mu);
        l = fmaf(w, q[1], l);
        sum = fmaf(w, q[2], sum);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = fmaf(w, x[s][i], o[i]);
      }
#pragma unroll
    for (int s = 0; s < 8; ++s)
      if (s0 + 8 + s < n) x[s] = *reinterpret_cast<const f32x4*>(src + (int64_t)(s0 + 8 + s) * rows * a.d);
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
  if (a.lse && c == 0) a.lse[(b * a.kvh * a.hg + head) * a.Nq + qi] = sum > 0.f ? (mu + log2f(sum)) * LN2 : -INFINITY;
}

struct Plan {
  bool resident;
  int nw, chk, nb, nsplit, lds;
};
// Resident keys while two blocks of them fit a CU (4 waves), or one block of 8 waves when there are query tiles for them: 48 x 4096
// queries, 8 heads of 40, 77 keys 98 us, streamed 102; 48 x 1024 queries, 8 heads of 80, 257 keys 54 against 74, 48 x 256 24 against 21.
// The blocks are as many as are resident at once.  Streamed with one wave per block when one tile holds all queries (64 x 1 query, 16
// heads of 64 on 2 key heads, 4097 keys: 36 us, four waves of which three wait 55), else four.  The keys are cut into parts while not
// even half the chip has a block, a part keeping at least 256 keys (the same call uncut 141 us, with twice the parts 42, with half of
// them 48; 2 x 1024 queries, 8 heads of 40, 4097 keys: 51, uncut 84, with twice the parts 39).
Plan plan(const Args& a) {
  Plan p{};
  const int ks = k_steps(a.d), cus = cu_count(), eg = a.Be * a.kvh;
  const int T = (a.R + 31) / 32, all = kv_lds(ks, (a.Nk + 63) / 64 * 64);
  p.nsplit = 1;
  if (all <= 80000 || (all <= 160000 && T >= 16)) {
    p.resident = true;
    p.nw = all <= 80000 ? 4 : 8;
    p.chk = 32;
    p.lds = all;
    const int most = (T + p.nw - 1) / p.nw, fit = 160000 / (all > 1000 ? all : 1000), per_cu = p.nw == 8 ? 1 : fit < 4 ? fit : 4;
    p.nb = (per_cu * cus + eg - 1) / eg;
    if (p.nb > most) p.nb = most;
    return p;
  }
  p.nw = T == 1 ? 1 : 4;
  p.chk = stream_keys(ks, p.nw);
  p.lds = 2 * kv_lds(ks, p.chk);
  p.nb = (T + p.nw - 1) / p.nw;
  const int64_t blocks = (int64_t)eg * p.nb, fill = p.nw == 1 ? 4 * cus : cus;
  if (2 * blocks <= fill) {
    int64_t n = fill / blocks;
    const int parts = (a.Nk + 255) / 256;
    if (n > parts) n = parts;
    p.nsplit = n > 64 ? 64 : n < 1 ? 1 : (int)n;
  }
  return p;
}

size_t ws_bytes(const Args& a, const Plan& p) {
  return p.nsplit > 1 ? (size_t)p.nsplit * a.Be * a.kvh * a.R * (a.d + 4) * sizeof(float) : 0;
}

template <int DT, int KS>
int launch(const Args& a, const Plan& p, hipStream_t st) {
  const dim3 grid((unsigned)(a.Be * a.kvh) * (unsigned)p.nb, (unsigned)p.nsplit);
  constexpr int CH1 = stream_keys(KS, 1), CH4 = stream_keys(KS, 4);
  if (p.resident && p.nw == 4) hipLaunchKernelGGL((xattn_kernel<DT, KS, true, 4, 32>), grid, dim3(256), p.lds, st, a);
  else if (p.resident) hipLaunchKernelGGL((xattn_kernel<DT, KS, true, 8, 32>), grid, dim3(512), p.lds, st, a);
  else if (p.nw == 1) hipLaunchKernelGGL((xattn_kernel<DT, KS, false, 1, CH1>), grid, dim3(64), p.lds, st, a);
  else hipLaunchKernelGGL((xattn_kernel<DT, KS, false, 4, CH4>), grid, dim3(256), p.lds, st, a);
  MIMO_LAUNCH_CHECK();
  if (p.nsplit > 1) {
    const int d4 = a.d / 4, per = 256 / d4 < 32 ? 256 / d4 : 32;
    const int64_t rows = (int64_t)a.Be * a.kvh * a.R;
    hipLaunchKernelGGL((xattn_join_kernel<DT>), dim3((unsigned)((rows + per - 1) / per)), dim3(256), 0, st, a);
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
  a.nb = pl.nb; a.nsplit = pl.nsplit; a.lag = fminf(LAG / a.c, 1e30f);
  if (ws_bytes(a, pl) > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < ws_bytes(a, pl))) return MIMO_EINVAL;
  a.ws = (float*)workspace;
  if (dtype == MIMO_F16) return dispatch<MIMO_F16>(a, pl, (hipStream_t)stream);
  if (dtype == MIMO_BF16) return dispatch<MIMO_BF16>(a, pl, (hipStream_t)stream);
  return MIMO_EDTYPE;
}
