// cross_attention_bwd.hip — gradients of the cross attention (gfx950, MFMA 32x32x16).
//
//   P = exp(scale q.k - lse), delta[q] = sum_d dO o O, dP = dO.V^T, dS = P (dP - delta)
//   dQ = scale dS.K          dK = scale dS^T.Q          dV = P^T.dO        (dK, dV: summed over every query that sees the key)
//
// Two kernels, both recompute P from lse (no score is ever stored):
//   xattn_dq_kernel   S^T = K.Q^T and dP^T = V.dO^T: a lane owns a query, dS^T packed is the operand of dQ^T = K^T.dS^T.  Keys
//                     resident in LDS as in the forward, or streamed; also leaves delta (few keys: sum_k P dP instead of dO.O).
//                     What bounds it: the rows of q, dO, O and dQ, a piece of 2 d bytes per head and row: 55 us for 16 x 4096 queries,
//                     8 heads of 40, 77 keys (3.1 TB/s); for 24 x 255 queries, 8 heads of 160, 257 streamed keys the exponentials and
//                     LDS reads between the products (35 us; a third of its blocks have no key there, so about one wave per SIMD).
//   xattn_dkv_kernel  S = Q.K^T and dP = dO.V^T: a lane owns a key, a wave 32 of them with K and V in registers; the block's waves
//                     share the query tiles that pass through LDS, P and dS packed are the operands of dV^T = dO^T.P and
//                     dK^T = Q^T.dS.  The flat rows are cut into parts (gridDim.y) when the keys do not fill the chip; their
//                     fp32 sums are joined in a fixed order by xattn_dkv_join_kernel: no atomics, the same bits every time.
// P and dS are rounded to the operand type for the last products (one rounding each, relative to the value, of the size of the results'
// own; dQ of heads up to 32 wide takes dS's remainder as well); sums, lse and delta are fp32.  In fp16 dS is lifted by a power of two
// first (lift_of), so that neither a small nor a large dO takes it out of that type's 30 binades.
// What bounds dk / dv: products (22 % of the time), LDS (32 %) and vector instructions (34 %) hardly overlap at two waves per SIMD: 47 to
// 49 us at the last of these shapes, 44 us at the first.
#include "cross_attention.hip.h"

namespace mimo_xattn {
namespace {

constexpr int stream_keys(int ks) { return ks >= 6 ? 32 : 64; }  // keys per streamed buffer of dq

// dS in fp16.  dS follows dO, which may be anything from 1e-6 (a mean over many rows) to the loss scale of its user, and P, which is about
// 1 / keys: unscaled it loses its bits below 2^-14 and is infinite above 65504, where dQ and dK, sums of it, still fit (512 rows, 1024
// keys, dO of 1e-3: dQ off by 1.7e-3 relative l2 instead of 6.5e-4).  |dP| <= d max|V| max|dO| and P <= 1, so f dS with f = 2^(15 - e), e the
// exponent of d max|V| max|dO| + |delta|, is always finite; a typical dP lies some seven binades below that bound, which leaves P 2^8 down
// to 2^-14.  dq takes f per query (its lane's), dk / dv one for all rows of a key head, from the largest e that dq's waves left; f comes
// off the fp32 sums exactly.  Price: max|V| while the keys are staged, max|dO| beside delta; nothing per pair of query and key (dQ with
// resident keys 55.5 us with and without, 16 x 4096 queries, 8 heads of 40, 77 keys; streamed 83 -> 89, 16 rows of 4097 keys of width 64,
// and 36.5 where bf16 takes 33.5, 24 x 255 queries, 8 heads of 160, 257 keys; a running maximum of |dS| in both kernels' inner loops
// added 10 us to the first shape's 139).
constexpr int NO_ROW = -1000;  // e of a wave without rows
__device__ __forceinline__ float lift_of(int e) { return ldexpf(1.f, 15 - e); }
// the largest of the wave's two packed maxima, left for the block in one of eight words behind the value rows, which no read of this
// file's kernels reaches (lane exchanges by DPP: through LDS they took 0.3 us per streamed chunk)
__device__ __forceinline__ void put_top(uint32_t top, uint32_t* slots, int lane, int wave) {
  uint32_t m = max(top & 0xffffu, top >> 16);
#define STEP(ctrl) m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, ctrl, 0xf, 0xf, false))
  STEP(0x111); STEP(0x112); STEP(0x114); STEP(0x118);  // row_shr 1 2 4 8
  STEP(0x142); STEP(0x143);                            // row_bcast 15 31
#undef STEP
  if (lane == 63) slots[wave] = m;
}
template <int NW>
__device__ __forceinline__ float get_top(const uint32_t* slots) {
  uint32_t m = 0u;
#pragma unroll
  for (int w = 0; w < NW; ++w) m = max(m, slots[w]);
  return HT<MIMO_F16>::to_f((uint16_t)__builtin_amdgcn_readfirstlane((int)m));
}

// RESIDENT: NW = 4 or 8 waves per block as in the forward; streamed: 4
template <int DT, int KS, bool RESIDENT, int NW>
__global__ __launch_bounds__(64 * NW, NW == 4 && KS <= 3 ? 3 : 2) void xattn_dq_kernel(const Args a) {
  constexpr int OT = (KS + 1) / 2, P = 16 * KS + 8, THREADS = 64 * NW, CH = stream_keys(KS);
  constexpr bool LIFT = DT == MIMO_F16;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h2 = lane >> 5, li = lane & 31;
  const unsigned L = xcd_remap(blockIdx.x, gridDim.x);
  const int g = (int)(L % (unsigned)a.kvh);
  const int e = (int)(L / (unsigned)a.kvh) % a.Be, j = (int)(L / (unsigned)a.kvh) / a.Be;
  const int len = valid_len(a, e);
  const int T = (a.R + 31) >> 5;
  const int npad = RESIDENT ? (a.Nk + 31) / 32 * 32 : CH, stride = kv_lds(KS, npad);
  auto ks_of = [&](int b) { return reinterpret_cast<uint16_t*>(smem + b * stride); };
  auto vs_of = [&](int b) { return reinterpret_cast<uint16_t*>(smem + b * stride) + npad * P; };
  auto bias_of = [&](int b) { return reinterpret_cast<float*>(smem + b * stride + 2 * npad * P * 2 + 64); };
  auto tops_of = [&](int b) { return reinterpret_cast<uint32_t*>(smem + b * stride + 2 * npad * P * 2); };
  Stager<KS, THREADS, CH> stager;
  stager.open(a, e, g);
  if constexpr (RESIDENT) {
    const uint32_t top = stage_all<DT, KS, THREADS, LIFT>(a, e, g, len, ks_of(0), vs_of(0), bias_of(0), false, tid);
    if constexpr (LIFT) put_top(top, tops_of(0), lane, wave);
    lds_barrier();
  }
  auto commit = [&](int b) {
    stager.top = 0u;
    stager.template commit<DT, LIFT>(a, ks_of(b), vs_of(b), bias_of(b), false, tid);
    if constexpr (LIFT) put_top(stager.top, tops_of(b), lane, wave);
  };
  const int step = a.nb * NW;
  int t = j * NW + wave;
  [[maybe_unused]] int most = NO_ROW;  // the largest e of the wave's rows (uniform)

  // delta from the rounded output is off by u |dO||O|: nothing beside dS where many keys share the row, but half of dQ's error where
  // two do (relative l2 of dQ at 2, 8, 32 keys of width 40 in fp16: 4.7, 3.2, 3.05e-4; from P and dP 2.9, 3.0, 2.96e-4).  Up to 32
  // keys that count are gathered into one tile for it, lane i (of each half) taking the i-th of them.
  int n_few = 0, mine = 0;
  for (int k = 0; k < len && n_few <= 32; k += 64) {
    const bool on = k + lane < len && (!a.mask || a.mask[(int64_t)e * a.smb + min(k + lane, len - 1)] != 0);
    const unsigned long long b = __builtin_amdgcn_ballot_w64(on);
    const int rank = n_few + (int)__builtin_amdgcn_mbcnt_hi((unsigned)(b >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)b, 0u));
    const int got = __builtin_amdgcn_ds_permute(4 * (on && rank < 32 ? rank : 63), on ? k + lane + 1 : 0);  // (lane 63 keeps the rest)
    if (lane < 32 && got > 0) mine = got - 1;
    n_few += __builtin_popcountll(b);
  }
  const bool few = n_few <= 32;
  mine = __shfl(mine, li, 64);

  struct Row {
    uint4 q[KS], d[KS], o[KS];
    float lse;
  };
  auto place = [&](int tt, int64_t& b, int& qi, int& head) {
    int img, hh;
    flat_row(a, min(32 * tt + li, a.R - 1), img, qi, hh);
    head = g * a.hg + hh;
    b = (int64_t)e * a.G + img;
  };
  auto request = [&](int tt, Row& r) {
    int64_t b;
    int qi, head;
    place(tt, b, qi, head);
    const int64_t col = (int64_t)head * a.d;
    load_row<KS>(r.d, a.dout + b * a.sdb + (int64_t)qi * a.sdr + col, a.d, h2);
    load_row<KS>(r.o, a.o + b * a.sob + (int64_t)qi * a.sor + col, a.d, h2);
    load_row<KS>(r.q, a.q + b * a.sqb + (int64_t)qi * a.sqr + col, a.d, h2);
    r.lse = a.lse_in[(b * a.kvh * a.hg + head) * a.Nq + qi];
  };
  // narrow heads: the next tile's rows are requested before this one's products (wider ones have no registers for that)
  constexpr bool AHEAD = RESIDENT && KS <= 5;
  Row nx;
  if (AHEAD && t < T) request(t, nx);

  // (streamed: one tile per wave, as in the forward)
  for (bool first = true; RESIDENT ? t < T : first; t += step, first = false) {
    uint4 qf[KS], df[KS];
    float delta = 0.f, l2;
    [[maybe_unused]] float size = 0.f;  // max |dO|
    {
      if constexpr (!AHEAD) request(min(t, T - 1), nx);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int kk = 16 * s + 8 * h2;
        float x[8], y[8];
        unpack8<DT>(nx.o[s], x);
        unpack8<DT>(nx.d[s], y);
        float p = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) p = fmaf(x[i], y[i], p);
        delta += kk < a.d ? p : 0.f;
        if constexpr (LIFT) {
#pragma unroll
          for (int i = 0; i < 8; ++i) size = fmaxf(size, __builtin_fabsf(y[i]));  // (channels behind the last one repeat the first)
        }
        qf[s] = nx.q[s];
        df[s] = nx.d[s];
      }
      l2 = nx.lse * LOG2E;
      if (AHEAD && t + step < T) request(t + step, nx);
      delta += __shfl_xor(delta, 32, 64);
      if constexpr (LIFT) size = fmaxf(size, __shfl_xor(size, 32, 64));
    }
    if (l2 == -INFINITY) l2 = INFINITY;  // a row without a key: P = exp2(0 - inf) = 0
    if (few) {
      const uint16_t* kp = a.k + (int64_t)e * a.skb + (int64_t)mine * a.skr + (int64_t)g * a.d;
      const uint16_t* vp = a.v + (int64_t)e * a.svb + (int64_t)mine * a.svr + (int64_t)g * a.d;
      f32x16 s, dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.f;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const int kk = 16 * i + 8 * h2;
        uint4 x = make_uint4(0, 0, 0, 0), y = x;
        if (li < n_few && kk < a.d) {
          x = *reinterpret_cast<const uint4*>(kp + kk);
          y = *reinterpret_cast<const uint4*>(vp + kk);
        }
        s = HT<DT>::mfma32(x, qf[i], s);
        dp = HT<DT>::mfma32(y, df[i], dp);
      }
      delta = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (8 * (r >> 2) + 4 * h2 + (r & 3) < n_few) delta = fmaf(fast_exp2(fmaf(s[r], a.c, -l2)), dp[r], delta);
      delta += __shfl_xor(delta, 32, 64);
    }
    const RowPlace out = row_place(a, e, g, min(t, T - 1), li, a.out, a.delta);
    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, delta), out.table, t < T && h2 == 0 ? out.stat : 0xF0000000u, 0, 0);
    f32x16 acc[OT];
#pragma unroll
    for (int i = 0; i < OT; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
    // e, f and f delta for values up to v_top; a streamed chunk that holds larger ones brings f, and the sums so far, down
    [[maybe_unused]] float v_top = -1.f;
    [[maybe_unused]] int ex = 15;
    float f = 1.f, off = delta;
    auto raise = [&](float top) {
      v_top = top;
      const float d1 = ldexpf(off, ex - 15);
      const int to = __builtin_amdgcn_frexp_expf(fmaf(size * (float)a.d, top, __builtin_fabsf(d1)));
      if constexpr (!RESIDENT) {
        const float by = ldexpf(1.f, ex - to);
#pragma unroll
        for (int i = 0; i < OT; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[i][r] *= by;
      }
      ex = to;
      f = lift_of(to);
      off = d1 * f;
    };
    if constexpr (LIFT && RESIDENT) raise(get_top<NW>(tops_of(0)));

    auto tile = [&](const uint16_t* ks, const uint16_t* vs, const float* bias, int kr, bool masked) {
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
      for (int r = 0; r < 16; ++r) s[r] = fast_exp2(fmaf(s[r], a.c, -l2)) * (LIFT ? fmaf(dp[r], f, -off) : dp[r] - off);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint4 ds = pack_k<DT>(s, u);
#pragma unroll
        for (int i = 0; i < OT; ++i) acc[i] = HT<DT>::mfma32(read_tr(ks, P, kr + 16 * u, 32 * i, lane), ds, acc[i]);
        if constexpr (KS == 2) {  // what dS lost, too: a narrow head's dQ is a sum that largely cancels (relative l2 at width 8, 77 keys
          float hi[8];            // in fp16: 3.3e-4 with dS rounded, 2.35e-4 with its remainder, the result's own rounding 2.1e-4)
          unpack8<DT>(ds, hi);
          const uint4 lo = make_uint4(pack2<DT>(s[8 * u] - hi[0], s[8 * u + 1] - hi[1]), pack2<DT>(s[8 * u + 2] - hi[2], s[8 * u + 3] - hi[3]),
                                      pack2<DT>(s[8 * u + 4] - hi[4], s[8 * u + 5] - hi[5]), pack2<DT>(s[8 * u + 6] - hi[6], s[8 * u + 7] - hi[7]));
          acc[0] = HT<DT>::mfma32(read_tr(ks, P, kr + 16 * u, 0, lane), lo, acc[0]);
        }
      }
    };
    if constexpr (RESIDENT) {
      for (int kr = 0; kr < len; kr += 32) tile(ks_of(0), vs_of(0), bias_of(0), kr, a.mask || kr + 32 > len);
    } else {
      const int chunks = (len + CH - 1) / CH;
      if (chunks > 0) {
        stager.issue(a, e, len, 0, tid);
        commit(0);
        settle<KS>(qf);
        settle<KS>(df);
        if (chunks > 1) stager.issue(a, e, len, CH, tid);
      }
      for (int i = 0; i < chunks; ++i) {
        lds_barrier();
        const int bf = i & 1;
        if constexpr (LIFT) {
          const float top = get_top<NW>(tops_of(bf));
          if (top > v_top) raise(top);
        }
        if (t < T) {
          tile(ks_of(bf), vs_of(bf), bias_of(bf), 0, a.mask || i * CH + 32 > len);
          if (CH > 32 && i * CH + 32 < len) tile(ks_of(bf), vs_of(bf), bias_of(bf), 32, a.mask || i * CH + 64 > len);
        }
        if (i + 1 < chunks) {
          commit(bf ^ 1);
          if (i + 2 < chunks) stager.issue(a, e, len, (i + 2) * CH, tid);
        }
      }
    }
    if (t >= T) continue;
    if constexpr (LIFT) {
      for (unsigned long long b = __builtin_amdgcn_ballot_w64(ex > most); b != 0ull; b = __builtin_amdgcn_ballot_w64(ex > most))
        most = __builtin_amdgcn_readlane(ex, (int)__builtin_ctzll(b));
    }
#pragma unroll
    for (int i = 0; i < OT; ++i) store_tile<DT>(acc[i], LIFT ? ldexpf(a.scale, ex - 15) : a.scale, out, i, a.d, h2);
  }
  if constexpr (LIFT) {
    if (a.tops && lane == 0) a.tops[((int64_t)e * a.kvh + g) * a.slots + j * NW + wave] = most;
  }
}

// query rows per LDS buffer: what a thread can hold on its way
constexpr int qt_rows(int ks, int nw) { return ks <= 4 && nw > 2 ? 64 : 32; }
constexpr int dkv_buffers(int ks, int nw) { return 2 * (2 * qt_rows(ks, nw) * (16 * ks + 8) * 2 + 2 * qt_rows(ks, nw) * 4 + 64); }
// waves that share a key tile: dK and dV of a wide head do not fit one wave's registers beside its K and V, so two waves form the
// same P and dS and each takes half of the channels (and V's fragments are in LDS): two waves per SIMD without spills, 55 us against
// 94 with one wave of 500 registers (24 x 255 queries, 8 heads of 160, 257 keys)
constexpr int dkv_share(int ks) { return ks >= 8 ? 2 : 1; }
constexpr int dkv_lds(int ks, int nw) { return dkv_buffers(ks, nw) + (dkv_share(ks) == 2 ? nw * ks * 1024 : 0); }
constexpr int dkv_occ(int ks) { return ks <= 2 ? 3 : 2; }    // waves per SIMD

// NW: key tiles of a block
template <int DT, int KS, int NW>
__global__ __launch_bounds__(64 * NW * dkv_share(KS), dkv_occ(KS)) void xattn_dkv_kernel(const Args a) {
  constexpr int OT = (KS + 1) / 2, P = 16 * KS + 8, SHARE = dkv_share(KS), OW = (OT + SHARE - 1) / SHARE, THREADS = 64 * NW * SHARE,
                QT = qt_rows(KS, NW);
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  constexpr int BUF = 2 * QT * P * 2 + 2 * QT * 4 + 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h2 = lane >> 5, li = lane & 31;
  const int part = SHARE == 1 ? 0 : wave & 1, o0 = part * OW;  // this wave's channel tiles: o0 .. o0 + OW (less one if OT is odd)
  // blocks of one XCD: the key heads of the same rows, then the key groups
  const unsigned L = xcd_remap(blockIdx.x, gridDim.x);
  const int g = (int)(L % (unsigned)a.kvh);
  const int e = (int)(L / (unsigned)a.kvh) % a.Be, kt = (int)(L / (unsigned)a.kvh) / a.Be;
  const int len = valid_len(a, e);
  const int key0 = (kt * NW + wave / SHARE) * 32, key = key0 + li;
  const bool valid = key_valid(a, e, len, min(key, a.Nk - 1)) && key < a.Nk;
  const bool any = key0 < len;  // (wave-uniform)
  // flat rows of this part, in whole QT tiles
  const int T = (a.R + QT - 1) / QT, per = (T + a.nsplit - 1) / a.nsplit;
  const int t_lo = min(T, (int)blockIdx.y * per), t_hi = kt * NW * 32 < len ? min(T, t_lo + per) : t_lo;

  uint4 kf[KS], vf[SHARE == 1 ? KS : 1];
  uint4* vl = reinterpret_cast<uint4*>(smem + dkv_buffers(KS, NW) + wave / SHARE * KS * 1024) + lane;  // SHARE == 2: [KS][64]
  {
    const uint16_t* kp = a.k + (int64_t)e * a.skb + (int64_t)(valid ? key : 0) * a.skr + (int64_t)g * a.d;
    const uint16_t* vp = a.v + (int64_t)e * a.svb + (int64_t)(valid ? key : 0) * a.svr + (int64_t)g * a.d;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int kk = 16 * s + 8 * h2;
      uint4 x = make_uint4(0, 0, 0, 0), y = x;
      if (valid && kk < a.d) {
        x = *reinterpret_cast<const uint4*>(kp + kk);
        y = *reinterpret_cast<const uint4*>(vp + kk);
      }
      kf[s] = x;
      if (SHARE == 1) vf[SHARE == 1 ? s : 0] = y;
      else if (part == 0) vl[64 * s] = y;
    }
  }
  f32x16 dk[OW], dv[OW];
#pragma unroll
  for (int i = 0; i < OW; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) dk[i][r] = dv[i][r] = 0.f;

  // rows [QT t, QT t + QT) of q and dO, their lse (log2 units) and delta: requested (issue), written to a buffer (commit).  Rows
  // behind the last one repeat it with lse = inf: P = 0.  Where there are eight threads to a row they take its 16-byte chunks, else
  // the chunks of the tile are dealt to the threads one after another; threads without one repeat the last: no request is behind a
  // branch.  The channels behind the last one are zeroed once.
  constexpr bool BY_ROW = THREADS >= 8 * QT && KS > 4;
  constexpr int NC = BY_ROW ? (2 * KS + 7) / 8 : (QT * 2 * KS + THREADS - 1) / THREADS;
  typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
  u32x4 xr[NC], yr[NC];
  float lr, dr;
  int place[NC];  // row << 8 | channel of this thread's chunks
  {
    const int dc = a.d >> 3;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = min(tid + i * THREADS, QT * dc - 1), row = BY_ROW ? min(tid >> 3, QT - 1) : (int)div_fast((uint32_t)c, a.by_dc);
      place[i] = row << 8 | (BY_ROW ? min((tid & 7) + 8 * i, dc - 1) : c - row * dc) * 8;
    }
    for (int c = tid; c < 2 * 2 * QT * (2 * KS - dc); c += THREADS) {  // (usually none)
      const int row = c / (2 * KS - dc), col = dc + c - row * (2 * KS - dc);  // rows of q, dO of buffer 0, then of buffer 1
      *reinterpret_cast<uint4*>(smem + (row >= 2 * QT ? BUF - 2 * QT * P * 2 : 0) + row * P * 2 + col * 16) = make_uint4(0, 0, 0, 0);
    }
  }
  // f of dS, from the largest e of this key head's rows; in fp16 P itself is held as 2^14 P, f is what dS needs beyond that: a key among
  // 16384 has P below fp16's normal range (64 queries, 60000 keys: dV off by 6.8e-4 relative l2 instead of 3e-4)
  constexpr int UP = DT == MIMO_F16 ? 14 : 0;
  float f = 1.f;
  if constexpr (DT == MIMO_F16) {
    const int* tops = a.tops + ((int64_t)e * a.kvh + g) * a.slots;
    int m = NO_ROW;
#pragma unroll 4
    for (int i = lane; i < a.slots; i += 64) m = max(m, tops[i]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = max(m, __shfl_xor(m, o, 64));
    f = lift_of(m + UP);
  }
  auto issue = [&](int t) __attribute__((always_inline)) {
    const uint16_t *qp = nullptr, *dp = nullptr;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      int at = place[i];
      asm volatile("" : "+v"(at));  // addresses are made anew for every tile: kept over the products they would cost registers
      if (!BY_ROW || i == 0) {
        int img, qi, hh;
        flat_row(a, min(t * QT + (at >> 8), a.R - 1), img, qi, hh);
        const int64_t bb = (int64_t)e * a.G + img, col = (int64_t)(g * a.hg + hh) * a.d;
        qp = a.q + bb * a.sqb + (int64_t)qi * a.sqr + col;
        dp = a.dout + bb * a.sdb + (int64_t)qi * a.sdr + col;
      }
      xr[i] = *reinterpret_cast<const u32x4*>(qp + (at & 255));
      yr[i] = *reinterpret_cast<const u32x4*>(dp + (at & 255));
    }
    static_assert(QT <= THREADS, "a thread per row");
    int img, qi, hh;
    flat_row(a, min(t * QT + (tid & (QT - 1)), a.R - 1), img, qi, hh);
    const int64_t stat = (((int64_t)e * a.G + img) * a.kvh * a.hg + g * a.hg + hh) * a.Nq + qi;
    lr = a.lse_in[stat];
    dr = a.delta[stat];
  };
  auto commit = [&](int t, int b) __attribute__((always_inline)) {
    uint16_t* qs = reinterpret_cast<uint16_t*>(smem + b * BUF);
    float* l2 = reinterpret_cast<float*>(smem + b * BUF + 2 * QT * P * 2 + 64);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      int at = place[i];
      asm volatile("" : "+v"(at));
      uint16_t* to = qs + (at >> 8) * P + (at & 255);
      *reinterpret_cast<u32x4*>(to) = xr[i];
      *reinterpret_cast<u32x4*>(to + QT * P) = yr[i];
    }
    float l = lr;
    asm volatile("" : "+v"(l));  // (not earlier: what is made of it would wait for the requests)
    if (tid < QT) {
      l2[tid] = l == -INFINITY || t * QT + tid >= a.R ? INFINITY : fmaf(l, LOG2E, (float)-UP);
      l2[QT + tid] = dr * f;
    }
  };
  // row tile t is in buffer (t - t_lo) & 1, t + 1 on its way
  if (t_lo < t_hi) {
    issue(t_lo);
    commit(t_lo, 0);
    settle<KS>(kf);
    if constexpr (SHARE == 1) settle<KS>(vf);
    issue(min(t_lo + 1, t_hi - 1));
  }
  for (int t = t_lo; t < t_hi; ++t) {
    const int b = (t - t_lo) & 1;
    lds_barrier();
    const uint16_t* qs = reinterpret_cast<const uint16_t*>(smem + b * BUF);
    const uint16_t* ds = qs + QT * P;
    const float* l2 = reinterpret_cast<const float*>(smem + b * BUF + 2 * QT * P * 2 + 64);
    if (any) {
#pragma unroll
    for (int q0 = 0; q0 < QT; q0 += 32) {
      f32x16 s, dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.f;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        s = HT<DT>::mfma32(*reinterpret_cast<const uint4*>(qs + (q0 + li) * P + 16 * i + 8 * h2), kf[i], s);
        dp = HT<DT>::mfma32(*reinterpret_cast<const uint4*>(ds + (q0 + li) * P + 16 * i + 8 * h2), SHARE == 1 ? vf[SHARE == 1 ? i : 0] : vl[64 * i], dp);
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const f32x4 l = *reinterpret_cast<const f32x4*>(l2 + q0 + 8 * c + 4 * h2);
        const f32x4 dl = *reinterpret_cast<const f32x4*>(l2 + QT + q0 + 8 * c + 4 * h2);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = fast_exp2(fmaf(s[4 * c + r], a.c, -l[r]));
          s[4 * c + r] = p;
          dp[4 * c + r] = p * (DT == MIMO_F16 ? fmaf(dp[4 * c + r], f, -dl[r]) : dp[4 * c + r] - dl[r]);
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint4 pf = pack_k<DT>(s, u), sf = pack_k<DT>(dp, u);
#pragma unroll
        for (int i = 0; i < OW; ++i) {
          if (OT % SHARE && i == OW - 1 && part) continue;
          dv[i] = HT<DT>::mfma32(read_tr(ds, P, q0 + 16 * u, 32 * (o0 + i), lane), pf, dv[i]);
          dk[i] = HT<DT>::mfma32(read_tr(qs, P, q0 + 16 * u, 32 * (o0 + i), lane), sf, dk[i]);
        }
      }
    }
    }
    // (read last in the previous round, which every wave has left; behind the last tile it is not read, but nothing leads around a request)
    commit(t + 1, b ^ 1);
    issue(min(t + 2, t_hi - 1));
  }
  if (key >= a.Nk) return;
  const float drop = ldexpf(1.f, -UP), unlift = a.scale * drop / f;
  const int64_t C = (int64_t)a.kvh * a.d, at = ((int64_t)e * a.Nk + key) * C + (int64_t)g * a.d, plane = (int64_t)a.Be * a.Nk * C;
#pragma unroll
  for (int i = 0; i < OW; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int d0 = 32 * (o0 + i) + 8 * c + 4 * h2;
      if (d0 >= a.d) continue;
      f32x4 x, y;  // a key that the mask drops has no gradient (its columns hold what zeros gave)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[r] = valid ? dk[i][4 * c + r] * unlift : 0.f;
        y[r] = valid ? dv[i][4 * c + r] * drop : 0.f;
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

// dk / dv = the sum of the parts: eight runs of them side by side (a block takes 32 pieces of four numbers), then the runs in order
template <int DT>
__global__ __launch_bounds__(256) void xattn_dkv_join_kernel(const float* ws, uint16_t* dk, uint16_t* dv, int64_t plane, int parts) {
  __shared__ f32x4 sums[8][32];
  const int64_t n4 = plane >> 2, i = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
  const int run = threadIdx.x >> 5, per = (parts + 7) / 8, p0 = run * per, p1 = min(parts, p0 + per);
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (i < 2 * n4) {
    const float* w = ws + 4 * i;
#pragma unroll 4
    for (int p = p0; p < p1; ++p) s += *reinterpret_cast<const f32x4*>(w + (int64_t)p * 2 * plane);
  }
  sums[run][threadIdx.x & 31] = s;
  lds_barrier();
  if (run || i >= 2 * n4) return;
#pragma unroll
  for (int r = 1; r < 8; ++r) s += sums[r][threadIdx.x];
  *reinterpret_cast<uint2*>(i < n4 ? dk + 4 * i : dv + 4 * (i - n4)) = make_uint2(pack2<DT>(s[0], s[1]), pack2<DT>(s[2], s[3]));
}

struct Plan {
  bool resident;
  int dq_nw, lds, nb;      // dq
  int nw, groups, nsplit;  // dk / dv
};
// key tiles per block: heads whose tiles take two waves have 2
constexpr int least_tiles = 2;
constexpr int most_tiles(int ks) { return dkv_share(ks) == 2 ? 2 : 4; }
// dq: as the forward, but all keys in one part (forward and backward of 16 x 4096 queries, 8 heads of 40, 77 keys: resident 136.5 us,
// streamed 134.7).  dk / dv: the number of key tiles per block (two to four) that leaves the fewest waves without one (same queries, 64
// keys: 124.5 us, four of them always 128.4; a block of one wave for 32 keys 116 against 108); the rows are cut into as many parts as
// fill the chip once with resident blocks, a part keeping at least four row tiles (77 keys: twice the parts 143 us, a third 170).
Plan plan(const Args& a) {
  Plan p{};
  const int ks = k_steps(a.d), cus = cu_count(), eg = a.Be * a.kvh;
  const int all = kv_lds(ks, (a.Nk + 63) / 64 * 64), tq = (a.R + 31) / 32;
  p.resident = all <= 80000 || (all <= 160000 && tq >= 16);
  p.dq_nw = p.resident && all > 80000 ? 8 : 4;
  p.lds = p.resident ? all : 2 * kv_lds(ks, stream_keys(ks));
  const int most = (tq + p.dq_nw - 1) / p.dq_nw, fit = 160000 / (all > 1000 ? all : 1000), per_cu = p.dq_nw == 8 ? 1 : fit < 4 ? fit : 4;
  p.nb = p.resident ? (per_cu * cus + eg - 1) / eg : most;
  if (p.nb > most) p.nb = most;
  const int tiles = a.Nk > 0 ? (a.Nk + 31) / 32 : 1;  // (without keys there is no dk / dv launch)
  p.nw = most_tiles(ks);
  for (int w = p.nw - 1; w >= least_tiles; --w)
    if ((tiles + w - 1) / w * w < (tiles + p.nw - 1) / p.nw * p.nw) p.nw = w;
  p.groups = (tiles + p.nw - 1) / p.nw;
  const int T = (a.R + qt_rows(ks, p.nw) - 1) / qt_rows(ks, p.nw);
  const int by_waves = 4 * dkv_occ(ks) / (p.nw * dkv_share(ks)), by_lds = 160000 / dkv_lds(ks, p.nw);
  int64_t n = (int64_t)(by_waves < by_lds ? by_waves : by_lds) * cus / ((int64_t)eg * p.groups);
  if (n > T / 4) n = T / 4;
  if (n > 256) n = 256;
  p.nsplit = n < 1 ? 1 : (int)n;
  return p;
}

// workspace: delta [B, heads, Nq], the exponents that dq leaves for dk / dv, then the parts' dk / dv
int64_t delta_floats(const Args& a) { return ((int64_t)a.Be * a.kvh * a.R + 3) / 4 * 4; }
int64_t top_floats(const Args& a, const Plan& p) { return a.Nk > 0 ? ((int64_t)a.Be * a.kvh * p.nb * p.dq_nw + 3) / 4 * 4 : 0; }
size_t ws_bytes(const Args& a, const Plan& p) {
  const int64_t parts = p.nsplit > 1 ? (int64_t)p.nsplit * 2 * a.Be * a.Nk * a.kvh * a.d : 0;
  return (size_t)(delta_floats(a) + top_floats(a, p) + parts) * sizeof(float);
}

template <int DT, int KS>
int launch(Args& a, const Plan& p, hipStream_t st) {
  const unsigned eg = (unsigned)(a.Be * a.kvh);
  a.nb = p.nb; a.nsplit = 1; a.slots = p.nb * p.dq_nw;
  if (p.resident && p.dq_nw == 8) hipLaunchKernelGGL((xattn_dq_kernel<DT, KS, true, 8>), dim3(eg * (unsigned)p.nb), dim3(512), p.lds, st, a);
  else if (p.resident) hipLaunchKernelGGL((xattn_dq_kernel<DT, KS, true, 4>), dim3(eg * (unsigned)p.nb), dim3(256), p.lds, st, a);
  else hipLaunchKernelGGL((xattn_dq_kernel<DT, KS, false, 4>), dim3(eg * (unsigned)p.nb), dim3(256), p.lds, st, a);
  MIMO_LAUNCH_CHECK();
  if (a.Nk == 0) return MIMO_OK;
  a.nb = p.groups; a.nsplit = p.nsplit;
  const dim3 grid(eg * (unsigned)p.groups, (unsigned)p.nsplit);
  const int shm = dkv_lds(KS, p.nw);
  if constexpr (dkv_share(KS) == 2) {
    hipLaunchKernelGGL((xattn_dkv_kernel<DT, KS, 2>), grid, dim3(256), shm, st, a);
  } else {
    if (p.nw == 2) hipLaunchKernelGGL((xattn_dkv_kernel<DT, KS, 2>), grid, dim3(128), shm, st, a);
    if (p.nw == 3) hipLaunchKernelGGL((xattn_dkv_kernel<DT, KS, 3>), grid, dim3(192), shm, st, a);
    if (p.nw == 4) hipLaunchKernelGGL((xattn_dkv_kernel<DT, KS, 4>), grid, dim3(256), shm, st, a);
  }
  MIMO_LAUNCH_CHECK();
  if (p.nsplit > 1) {
    const int64_t plane = (int64_t)a.Be * a.Nk * a.kvh * a.d;
    hipLaunchKernelGGL((xattn_dkv_join_kernel<DT>), dim3((unsigned)((plane / 2 + 31) / 32)), dim3(256), 0, st, a.ws, a.dk, a.dv, plane,
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
  a.tops = a.Nk > 0 ? (int*)workspace + delta_floats(a) : nullptr;
  a.ws = (float*)workspace + delta_floats(a) + top_floats(a, pl);
  if (dtype == MIMO_F16) return dispatch<MIMO_F16>(a, pl, (hipStream_t)stream);
  if (dtype == MIMO_BF16) return dispatch<MIMO_BF16>(a, pl, (hipStream_t)stream);
  return MIMO_EDTYPE;
}
