// adapter.hip — low-rank adapters of many requests beside a shared projection, and their gradients (gfx950).
//
//   out[m] = a[m].W^T + bias + residual[m] + u[m].up[i]^T,   u[m] = scale[i] a[m].down[i]^T,   i = index[m / rows_per_index]
//
// The shared projection is one GEMM over all rows, whatever their adapters; u is a thin product in front of it (adapter_low_*:
// it reads `a` once, a stream) and u.up^T is added to the accumulators of the GEMM's tiles before their epilogue
// (tile_adapter): the result is written once and no intermediate is wider than the rank.  A tile walks the DISTINCT adapters of
// its rows, usually one; a row never takes part in another row's adapter (values are selected, not multiplied by zero, so a NaN
// in one adapter stays in its requests).
// u is kept as one rounded 16-bit value where the result is 16 bit, and as PLANES of 16-bit values (value | remainder: fp16 2, bf16
// 3, i.e. at least 22 mantissa bits) where the result is fp32 or gradients are to be taken: [M, planes rank].  A 16-bit result takes the
// value plane alone, da that of t: one rounding of the low-rank part, which is usually the smaller one, beside the result's own (out and
// da 2.27e-4 relative l2 in fp16, the result's rounding 2.08e-4; bf16 1.82e-3 and 1.66e-3; where the low-rank part is
// nearly all of it 2.94e-4).  In fp16 u and t end at 65504: beyond it the row's out or da, and the adapter's gradient, are infinite or NaN, as they are
// for any 16-bit value between two products.
//
// Backward of the same call, W frozen: t[m] = scale[i] dy[m].up[i];  da = dy.W + t.down (the same kernels on W^T and transposed
// adapters);  ddown[i] = sum_m t[m]^T a[m];  dup[i] = sum_m dy[m]^T u[m] (adapter_outer_kernel: rows stream through LDS, both
// operands by transposed reads; parts of the rows joined in a fixed order, no atomics).
#include "gemm_core.hip.h"

namespace {

inline int cu_count() {
  static const int cus = [] {
    int dev = 0, n = 0;
    if (hipGetDevice(&dev) != hipSuccess ||
        hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
    return n;
  }();
  return cus;
}
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

constexpr int planes_of(int dt) { return dt == MIMO_F16 ? 2 : 3; }
// on the remainder plane of t in fp16: gradients are small, 2^-25 is not small beside them (dO of 1e-5: ddown off by 4e-7; da, which takes
// the value alone, 1.58e-3, its own rounding 1.54e-3)
constexpr float T_SCALE = 2048.f;

// which adapter a row has
struct Rows {
  const int* index;
  int64_t M;
  unsigned rpi;
  int n;
};
__device__ __forceinline__ int adapter_of(const Rows& r, int64_t m) {
  if (m >= r.M) return -1;
  const int i = r.index[r.rpi == 1u ? (unsigned)m : (unsigned)m / r.rpi];
  return (unsigned)i < (unsigned)r.n ? i : -1;
}

// the adapter of the first row that is still to do (rows: `n` per-lane values, done or none = -1), or -1
template <int N>
__device__ __forceinline__ int next_adapter(const int (&ad)[N]) {
  int cur = -1;
#pragma unroll
  for (int i = N - 1; i >= 0; --i) {
    const unsigned long long b = __builtin_amdgcn_ballot_w64(ad[i] >= 0);
    if (b != 0ull) cur = __builtin_amdgcn_readlane(ad[i], (int)__builtin_ctzll(b));
  }
  return cur;
}

struct LowArgs {
  const uint16_t *X, *down;  // [M, ldx], [n, r, K]
  const float* scale;        // [n] or null
  uint16_t* low;             // [M, planes r]
  int64_t ldx;
  Rows rows;
  int K, r, planes;
  float lo_scale;            // a power of two on the remainder plane (fp16: small values keep their precision)
};

// the planes of four consecutive ranks of a row
template <int DT>
__device__ __forceinline__ void store_planes(const LowArgs& a, uint16_t* p, f32x4 v) {
  float scale = a.lo_scale;
  for (int q = 0;; ++q) {
    const uint2 h = make_uint2(pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]));
    *reinterpret_cast<uint2*>(p + q * a.r) = h;
    if (q + 1 >= a.planes) break;
    v[0] = (v[0] - HT<DT>::to_f((uint16_t)(h.x & 0xffffu))) * scale;
    v[1] = (v[1] - HT<DT>::to_f((uint16_t)(h.x >> 16))) * scale;
    v[2] = (v[2] - HT<DT>::to_f((uint16_t)(h.y & 0xffffu))) * scale;
    v[3] = (v[3] - HT<DT>::to_f((uint16_t)(h.y >> 16))) * scale;
    scale = 1.f;
  }
}

__device__ __forceinline__ float scale_of(const LowArgs& a, int ad) { return ad < 0 ? 0.f : a.scale ? a.scale[ad] : 1.f; }

// u for rows by the 32 (MFMA 16x16x32, down as the row operand: a lane ends with four consecutive ranks of one row).  A wave takes
// pieces of 64 channels: eight neighbouring lanes read 128 bytes of a row of X (of down), the piece passes through the wave's own
// LDS patch into fragments, the next piece is on its way meanwhile — fragments straight from memory (a row per lane) cost the
// address path a look-up per lane.  KSPLIT: the block's waves share 32 rows and take pieces in turn, joined in LDS in wave order —
// few rows; else each of four waves has 32 rows of its own.  Bound by the stream of X, down comes from L2: M = 196608, K = 320 in
// 22.5 us where X is in the last-level cache (5.6 TB/s), 40 us from HBM behind other traffic.
constexpr int low_waves(int rt, bool ksplit) { return ksplit && rt < 8 ? 8 : 4; }
template <int DT, int RT, bool KSPLIT>
__global__ __launch_bounds__(64 * low_waves(RT, KSPLIT)) void adapter_low_kernel(const LowArgs a) {
  constexpr int NW = low_waves(RT, KSPLIT), P = 72, PATCH = (32 + 16 * RT) * P;  // pitch: an odd number of 16-byte units
  constexpr int BYTES = NW * PATCH * 2, PART = KSPLIT ? NW * RT * 2 * 64 * 16 : 0;
  __shared__ __attribute__((aligned(16))) unsigned char smem[BYTES > PART ? BYTES : PART];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lg = lane >> 4, li = lane & 15, row0 = lane >> 3, c8 = (lane & 7) * 8;
  uint16_t* const xs = reinterpret_cast<uint16_t*>(smem) + wave * PATCH;
  uint16_t* const dsm = xs + 32 * P;
  const int64_t m0 = KSPLIT ? (int64_t)blockIdx.x * 32 : ((int64_t)blockIdx.x * 4 + wave) * 32;
  if (m0 >= a.rows.M) return;
  int ad[2], todo[2];
#pragma unroll
  for (int mi = 0; mi < 2; ++mi) ad[mi] = todo[mi] = adapter_of(a.rows, m0 + 16 * mi + li);
  const int pieces = (a.K + 63) / 64, first = KSPLIT ? wave : 0, way = KSPLIT ? NW : 1;
  uint4 xr[4], dr[2 * RT];
  auto request = [&](int p, int cur) {
    const int k = 64 * p + c8;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t m = m0 + row0 + 8 * i;
      xr[i] = make_uint4(0, 0, 0, 0);
      if (k < a.K && m < a.rows.M) xr[i] = *reinterpret_cast<const uint4*>(a.X + m * a.ldx + k);
    }
#pragma unroll
    for (int i = 0; i < 2 * RT; ++i) {
      const int j = row0 + 8 * i;
      dr[i] = make_uint4(0, 0, 0, 0);
      if (k < a.K && j < a.r) dr[i] = *reinterpret_cast<const uint4*>(a.down + ((int64_t)cur * a.r + j) * a.K + k);
    }
  };
  f32x4 res[RT][2];
#pragma unroll
  for (int t = 0; t < RT; ++t) res[t][0] = res[t][1] = (f32x4){0.f, 0.f, 0.f, 0.f};
  for (int cur = next_adapter<2>(todo); cur >= 0; cur = next_adapter<2>(todo)) {
    f32x4 acc[RT][2];
#pragma unroll
    for (int t = 0; t < RT; ++t) acc[t][0] = acc[t][1] = (f32x4){0.f, 0.f, 0.f, 0.f};
    if (first < pieces) request(first, cur);
    for (int p = first; p < pieces; p += way) {
      // LDS operations of a wave are carried out in order; the fences keep the compiler from reordering what other lanes wrote
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(xs + (row0 + 8 * i) * P + c8) = xr[i];
#pragma unroll
      for (int i = 0; i < 2 * RT; ++i) *reinterpret_cast<uint4*>(dsm + (row0 + 8 * i) * P + c8) = dr[i];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (p + way < pieces) request(p + way, cur);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint4 fx[2];
#pragma unroll
        for (int mi = 0; mi < 2; ++mi) fx[mi] = *reinterpret_cast<const uint4*>(xs + (16 * mi + li) * P + 32 * h + 8 * lg);
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          const uint4 fa = *reinterpret_cast<const uint4*>(dsm + (16 * t + li) * P + 32 * h + 8 * lg);
#pragma unroll
          for (int mi = 0; mi < 2; ++mi) acc[t][mi] = HT<DT>::mfma16(fa, fx[mi], acc[t][mi]);
        }
      }
      __builtin_amdgcn_wave_barrier();
    }
#pragma unroll
    for (int mi = 0; mi < 2; ++mi) {
      const bool mine = todo[mi] == cur;
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) res[t][mi][i] = mine ? acc[t][mi][i] : res[t][mi][i];
      todo[mi] = mine ? -1 : todo[mi];
    }
  }
  if constexpr (KSPLIT) {
    f32x4* const part = reinterpret_cast<f32x4*>(smem);
    lds_barrier();  // the patches are read
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int mi = 0; mi < 2; ++mi) part[((wave * RT + t) * 2 + mi) * 64 + lane] = res[t][mi];
    lds_barrier();
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int mi = 0; mi < 2; ++mi) {
        if ((2 * t + mi) % NW != wave) continue;  // (each wave finishes its share of the tiles)
        f32x4 v = part[(t * 2 + mi) * 64 + lane];
#pragma unroll
        for (int w = 1; w < NW; ++w) v += part[((w * RT + t) * 2 + mi) * 64 + lane];
        res[t][mi] = v;
      }
  }
#pragma unroll
  for (int mi = 0; mi < 2; ++mi) {
    const int64_t m = m0 + 16 * mi + li;
    const float sc = scale_of(a, ad[mi]);
    if (m >= a.rows.M) continue;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      if (KSPLIT && (2 * t + mi) % NW != wave) continue;
      const int j = 16 * t + 4 * lg;
      if (j >= a.r) continue;
      f32x4 v = res[t][mi] * sc;
      if (ad[mi] < 0) v = (f32x4){0.f, 0.f, 0.f, 0.f};
      store_planes<DT>(a, a.low + m * a.planes * a.r + j, v);
    }
  }
}

// u for rows that each have an adapter of their own: one block per row, a wave per four ranks in turn, lanes along K
template <int DT>
__global__ __launch_bounds__(256) void adapter_low_row_kernel(const LowArgs a) {
  const int64_t m = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int ad = adapter_of(a.rows, m);
  const float sc = scale_of(a, ad);
  const uint16_t* x = a.X + m * a.ldx;
  for (int j = 4 * wave; j < a.r; j += 16) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (ad >= 0) {
      const uint16_t* dn = a.down + ((int64_t)ad * a.r + j) * a.K;
#pragma unroll 3
      for (int k = 8 * lane; k < a.K; k += 512) {
        float p[8], q[8];
        unpack8<DT>(*reinterpret_cast<const uint4*>(x + k), p);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          unpack8<DT>(*reinterpret_cast<const uint4*>(dn + (int64_t)n * a.K + k), q);
#pragma unroll
          for (int i = 0; i < 8; ++i) s[n] = fmaf(p[i], q[i], s[n]);
        }
      }
#pragma unroll
      for (int n = 0; n < 4; ++n) s[n] = wave_sum(s[n]) * sc;
    }
    if (lane == 0) store_planes<DT>(a, a.low + m * a.planes * a.r + j, s);
  }
}

// [n, R, C] -> [n, C, R] of two stacks in one launch (blockIdx.z = which): 32 x 32 tiles through LDS
struct TransposeArgs {
  const uint16_t* in[2];
  uint16_t* out[2];
  int R[2], C[2];
};
__global__ __launch_bounds__(256) void adapter_transpose_kernel(const TransposeArgs a) {
  __shared__ uint16_t tile[32][33];
  const int z = blockIdx.z, R = a.R[z], C = a.C[z];
  const int tc = (C + 31) / 32, tr = (R + 31) / 32;
  const uint16_t* in = a.in[z] + (int64_t)blockIdx.y * R * C;
  uint16_t* out = a.out[z] + (int64_t)blockIdx.y * R * C;
  for (int t = blockIdx.x; t < tc * tr; t += gridDim.x) {
    const int r0 = t / tc * 32, c0 = t % tc * 32, x = threadIdx.x & 31, y = threadIdx.x >> 5;
    for (int i = y; i < 32; i += 8)
      if (r0 + i < R && c0 + x < C) tile[i][x] = in[(int64_t)(r0 + i) * C + c0 + x];
    lds_barrier();
    for (int i = y; i < 32; i += 8)
      if (c0 + i < C && r0 + x < R) out[(int64_t)(c0 + i) * R + r0 + x] = tile[x][i];
    lds_barrier();
  }
}

// sum over the rows of adapter blockIdx.y of low[m]^T x[m], for two pairs in one launch: (t, a) -> ddown and (u, dy) -> dup.
// A block owns 128 columns of x and all ranks; tiles of 64 rows pass through LDS row-major, both operands are read transposed
// (a row that is not this adapter's is staged as zeros on BOTH sides); the planes of low meet the same columns (fp16: the remainder
// plane has accumulators of its own, its scale comes off at the end).  Rows: only [first, last] of the adapter, cut into gridDim.z parts.
// Where an adapter's rows lie together it is bound by the streams of a and dy: 49152 rows of 640 + 640, r = 32 in 33 us (3.8 TB/s).
// Every row BETWEEN an adapter's first and last passes, its own or not, so adapters in turn read them again for each (the whole backward
// of the same rows, eight adapters: in runs of 6144 rows 115 us, 1024 rows of each in turn 228, an adapter per row in turn 339, in
// runs 132: with an index per row each block walks all of it first, 255 us against 194 at 200000 rows of 320 + 320).
struct OuterArgs {
  const uint16_t *x[2], *low[2];
  float* part[2];  // [parts][n][r][C]
  int64_t ldx[2];
  int C[2];
  float lo_scale[2];  // what the remainder plane has to be multiplied with
  Rows rows;
  int r, ct0;      // ct0: column tiles of the first pair
  FastDiv by_rpi, by_lc;
};

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
// operand of a 16x16x32 MFMA whose contraction index runs over LDS rows [r0, r0 + 32): lane (lg, i) gets column c0 + i of rows
// r0 + 8 lg .. + 8
__device__ __forceinline__ uint4 read_tr16(const uint16_t* tile, int pitch, int r0, int c0, int lane) {
  const int m = lane & 15, lg = lane >> 4;
  const uint16_t* p = tile + (r0 + 8 * lg + (m >> 2)) * pitch + c0 + 4 * (m & 3);
  const uint2 a = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)p));
  const uint2 b = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(p + 4 * pitch)));
  return make_uint4(a.x, a.y, b.x, b.y);
}

template <int DT, int RT>
__global__ __launch_bounds__(256) void adapter_outer_kernel(const OuterArgs a) {
  constexpr int NP = planes_of(DT), NA = DT == MIMO_F16 ? 2 : 1;
  constexpr int MR = 64, XP = 128 + 8, LP = NP * 16 * RT + 8;
  constexpr int NX = 4, NL = (NP * RT + 1) / 2;  // 16-byte chunks a thread stages per tile
  __shared__ __attribute__((aligned(16))) uint16_t xs[MR * XP];
  __shared__ __attribute__((aligned(16))) uint16_t ls[MR * LP];
  __shared__ int range[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 15, lg = lane >> 4;
  const int z = (int)blockIdx.x >= a.ct0;
  const int c0 = ((int)blockIdx.x - (z ? a.ct0 : 0)) * 128, C = a.C[z], who = blockIdx.y;
  // rows of this adapter
  if (tid == 0) {
    range[0] = 0x7fffffff;
    range[1] = -1;
  }
  lds_barrier();
  const int64_t G = (a.rows.M + a.rows.rpi - 1) / a.rows.rpi;
  int lo = 0x7fffffff, hi = -1;
  for (int64_t i0 = tid; i0 < G; i0 += 256 * 8) {
    int v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = i0 + 256 * u < G ? a.rows.index[i0 + 256 * u] : -1;
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (v[u] == who) {
        const int i = (int)i0 + 256 * u;
        lo = lo < i ? lo : i;
        hi = i;
      }
  }
  if (hi >= 0) {
    atomicMin(&range[0], lo);
    atomicMax(&range[1], hi);
  }
  for (int i = tid; i < MR * LP / 2; i += 256) reinterpret_cast<uint32_t*>(ls)[i] = 0u;  // columns behind the planes are never staged
  lds_barrier();
  f32x4 acc[NA][RT][2];
#pragma unroll
  for (int p = 0; p < NA; ++p)
#pragma unroll
    for (int t = 0; t < RT; ++t) acc[p][t][0] = acc[p][t][1] = (f32x4){0.f, 0.f, 0.f, 0.f};
  if (range[1] >= 0) {
    const int64_t m_lo = (int64_t)range[0] * a.rows.rpi;
    int64_t m_hi = ((int64_t)range[1] + 1) * a.rows.rpi;
    if (m_hi > a.rows.M) m_hi = a.rows.M;
    const int64_t tiles = (m_hi - m_lo + MR - 1) / MR, per = (tiles + gridDim.z - 1) / gridDim.z;
    const int64_t t_lo = blockIdx.z * per, t_hi = t_lo + per < tiles ? t_lo + per : tiles;
    const int lc = NP * a.r / 8;  // 16-byte chunks of a row of low
    // a tile on its way.  No branch and no dependent load between the requests: rows behind the last one repeat it, columns behind
    // the last one the first; `raw` = the index entry of row lane, it selects when the rows are written
    typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
    struct Piece {
      u32x4 x[NX], l[NL];
      int raw;
      int64_t m0;
    };
    auto fetch = [&](Piece& q, int64_t t) {
      int id0 = tid;
      asm volatile("" : "+v"(id0));
      const int64_t m0 = q.m0 = m_lo + t * MR;
      const int left = (int)(m_hi - m0 < MR ? m_hi - m0 : MR) - 1;
      const int c = c0 + (id0 & 15) * 8;
      const uint16_t* x = a.x[z] + m0 * a.ldx[z] + (c < C ? c : 0);
      const uint16_t* l = a.low[z] + m0 * NP * a.r;
#pragma unroll
      for (int i = 0; i < NX; ++i) q.x[i] = *reinterpret_cast<const u32x4*>(x + min((id0 >> 4) + 16 * i, left) * a.ldx[z]);
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int id = id0 + 256 * i, row = (int)div_fast(id, a.by_lc);
        q.l[i] = *reinterpret_cast<const u32x4*>(l + min(row, left) * NP * a.r + (id - row * lc) * 8);
      }
      const unsigned m = (unsigned)m0 + min(lane, left);
      q.raw = a.rows.index[div_fast(m, a.by_rpi)];
    };
    auto use = [&](const Piece& q) {
      int id0 = tid;
      asm volatile("" : "+v"(id0));
      const unsigned long long live = __builtin_amdgcn_ballot_w64(q.raw == who && q.m0 + lane < m_hi);
      lds_barrier();
#pragma unroll
      for (int i = 0; i < NX; ++i) {
        const int row = (id0 >> 4) + 16 * i;
        *reinterpret_cast<u32x4*>(xs + row * XP + (id0 & 15) * 8) = (live >> row) & 1 ? q.x[i] : (u32x4){0u, 0u, 0u, 0u};
      }
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int id = id0 + 256 * i, row = (int)div_fast(id, a.by_lc);
        if (row < MR) *reinterpret_cast<u32x4*>(ls + row * LP + (id - row * lc) * 8) = (live >> row) & 1 ? q.l[i] : (u32x4){0u, 0u, 0u, 0u};
      }
      lds_barrier();
    };
    auto products = [&]() {
#pragma unroll
      for (int k0 = 0; k0 < MR; k0 += 32) {
        uint4 fx[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) fx[c] = read_tr16(xs, XP, k0, wave * 32 + 16 * c, lane);
#pragma unroll
        for (int q = 0; q < RT; ++q) {
#pragma unroll
          for (int p = 0; p < NP; ++p) {
            const uint4 fl = read_tr16(ls, LP, k0, p * a.r + 16 * q, lane);
#pragma unroll
            for (int c = 0; c < 2; ++c) acc[p % NA][q][c] = HT<DT>::mfma16(fl, fx[c], acc[p % NA][q][c]);
          }
        }
      }
    };
    // the next tile on its way while this one's products run (two ahead were no faster: 121.9 against 117.5 us for the whole backward
    // at M = 49152, N = K = 640, r = 32, 48.7 against 47.3 us at 5003 x 640 x 1280, r = 24)
    if (t_lo < t_hi) {
      Piece q;
      fetch(q, t_lo);
      for (int64_t t = t_lo; t < t_hi; ++t) {
        use(q);
        fetch(q, t + 1 < t_hi ? t + 1 : t);  // (the last one again rather than a way around the request)
        products();
      }
    }
  }
  // lane: column c0 + .. + li, ranks 16 q + 4 lg + i
  float* out = a.part[z] + ((int64_t)blockIdx.z * gridDim.y + who) * a.r * C;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int col = c0 + wave * 32 + 16 * c + li;
    if (col >= C) continue;
#pragma unroll
    for (int q = 0; q < RT; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = 16 * q + 4 * lg + i;
        if (j < a.r) out[(int64_t)j * C + col] = NA == 1 ? acc[0][q][c][i] : fmaf(acc[NA - 1][q][c][i], a.lo_scale[z], acc[0][q][c][i]);
      }
  }
}

// the sum of the parts: eight runs of them side by side (a block takes 32 pieces of four columns), then the runs in order; ddown
// [n, r, K] as it lies, dup [n, N, r] transposed
__global__ __launch_bounds__(256) void adapter_join_kernel(const float* p0, const float* p1, float* ddown, float* dup, int n, int r, int K,
                                                           int N, int parts) {
  __shared__ f32x4 sums[8][32];
  const int64_t s0 = (int64_t)n * r * K, s1 = (int64_t)n * r * N, i = ((int64_t)blockIdx.x * 32 + (threadIdx.x & 31)) * 4;
  const int run = threadIdx.x >> 5, per = (parts + 7) / 8, q0 = run * per, q1 = min(parts, q0 + per);
  const bool first = i < s0;
  const int64_t at = first ? i : i - s0, plane = first ? s0 : s1;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (i < s0 + s1) {
    const float* p = (first ? p0 : p1) + at;
#pragma unroll 4
    for (int q = q0; q < q1; ++q) s += *reinterpret_cast<const f32x4*>(p + (int64_t)q * plane);
  }
  sums[run][threadIdx.x & 31] = s;
  lds_barrier();
  if (run || i >= s0 + s1) return;
#pragma unroll
  for (int u = 1; u < 8; ++u) s += sums[u][threadIdx.x];
  if (first) {
    *reinterpret_cast<f32x4*>(ddown + at) = s;
  } else {
    const int64_t row = at / N, c = at - row * N;  // row: (adapter, rank)
    float* o = dup + (row / r * N + c) * r + row % r;
#pragma unroll
    for (int k = 0; k < 4; ++k) o[(int64_t)k * r] = s[k];
  }
}

// A few rows (M <= 16 MG) against the whole weight: a block of eight waves takes 16 columns, the waves share K (every eighth
// k-step) and meet in LDS in wave order.  Bound by latency: one trip to W, one to the adapters (8 rows, N = K = 1280: 7.0 us, and 7.5
// for u in front of it, operands in no cache).  RT > 0 (MG = 1): u is computed
// here too, by every block for itself — the rows' down weights come from L2 and a launch is saved; RT = 0: u is given.
struct SkinnyArgs {
  const uint16_t *X, *W, *down, *up;
  const float *scale, *bias;
  const void* res;
  void* out;
  uint16_t* low;
  int64_t ldx, ldo, ldr;
  Rows rows;
  int N, K, r, planes, cols;  // cols: columns of low that take part (planes r for a fp32 result, else r)
  unsigned flags;
};
template <int DT, int MG, int RT>
__global__ __launch_bounds__(512) void adapter_skinny_kernel(const SkinnyArgs a) {
  constexpr int ULP = 3 * 16 * (RT > 0 ? RT : 1) + 8;
  __shared__ f32x4 part[8][MG + RT][64];
  __shared__ __attribute__((aligned(16))) uint16_t us[RT > 0 ? 16 * ULP : 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lg = lane >> 4, li = lane & 15, n0 = blockIdx.x * 16;
  int ad[MG];
  const uint16_t* x[MG];
#pragma unroll
  for (int g = 0; g < MG; ++g) {
    const int64_t m = 16 * g + li;
    x[g] = a.X + (m < a.rows.M ? m : 0) * a.ldx;
    ad[g] = adapter_of(a.rows, m);
  }
  const uint16_t* w = a.W + (int64_t)(n0 + li < a.N ? n0 + li : 0) * a.K;
  const int steps = (a.K + 31) / 32;
  f32x4 acc[MG];
#pragma unroll
  for (int g = 0; g < MG; ++g) acc[g] = (f32x4){0.f, 0.f, 0.f, 0.f};
  constexpr int UB = MG == 1 ? 5 : 3;
  for (int s0 = wave; s0 < steps; s0 += 8 * UB) {
    uint4 fw[UB], fx[UB][MG];
#pragma unroll
    for (int b = 0; b < UB; ++b) {
      const int kk = 32 * (s0 + 8 * b) + 8 * lg;
      fw[b] = make_uint4(0, 0, 0, 0);
      if (kk < a.K) fw[b] = *reinterpret_cast<const uint4*>(w + kk);
#pragma unroll
      for (int g = 0; g < MG; ++g) {
        fx[b][g] = make_uint4(0, 0, 0, 0);
        if (kk < a.K) fx[b][g] = *reinterpret_cast<const uint4*>(x[g] + kk);
      }
    }
#pragma unroll
    for (int b = 0; b < UB; ++b)
#pragma unroll
      for (int g = 0; g < MG; ++g) acc[g] = HT<DT>::mfma16(fw[b], fx[b][g], acc[g]);
  }
  if constexpr (RT > 0) {
    f32x4 u[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) u[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    int todo[1] = {ad[0]};
    for (int cur = next_adapter<1>(todo); cur >= 0; cur = next_adapter<1>(todo)) {
      const uint16_t* dn = a.down + (int64_t)cur * a.r * a.K;
      f32x4 v[RT];
#pragma unroll
      for (int t = 0; t < RT; ++t) v[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
      for (int s0 = wave; s0 < steps; s0 += 8 * UB) {
        uint4 fd[UB][RT], fx[UB];
#pragma unroll
        for (int b = 0; b < UB; ++b) {
          const int kk = 32 * (s0 + 8 * b) + 8 * lg;
          fx[b] = make_uint4(0, 0, 0, 0);
          if (kk < a.K) fx[b] = *reinterpret_cast<const uint4*>(x[0] + kk);
#pragma unroll
          for (int t = 0; t < RT; ++t) {
            fd[b][t] = make_uint4(0, 0, 0, 0);
            if (kk < a.K && 16 * t + li < a.r) fd[b][t] = *reinterpret_cast<const uint4*>(dn + (int64_t)(16 * t + li) * a.K + kk);
          }
        }
#pragma unroll
        for (int b = 0; b < UB; ++b)
#pragma unroll
          for (int t = 0; t < RT; ++t) v[t] = HT<DT>::mfma16(fd[b][t], fx[b], v[t]);
      }
      const bool mine = todo[0] == cur;
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) u[t][i] = mine ? v[t][i] : u[t][i];
      todo[0] = mine ? -1 : todo[0];
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) part[wave][MG + t][lane] = u[t];
  }
#pragma unroll
  for (int g = 0; g < MG; ++g) part[wave][g][lane] = acc[g];
  lds_barrier();
  // wave t < RT finishes rank tile t, then wave g of the first MG finishes row group g
  if constexpr (RT > 0) {
    if (wave < RT) {
      f32x4 v = part[0][MG + wave][lane];
#pragma unroll
      for (int q = 1; q < 8; ++q) v += part[q][MG + wave][lane];
      const int j = 16 * wave + 4 * lg;
      if (j < a.r) {
        const LowArgs la{nullptr, nullptr, a.scale, nullptr, 0, a.rows, 0, a.r, a.planes, 1.f};
        v *= scale_of(la, ad[0]);
        if (ad[0] < 0) v = (f32x4){0.f, 0.f, 0.f, 0.f};
        store_planes<DT>(la, us + li * ULP + j, v);
        if (blockIdx.x == 0 && li < a.rows.M) store_planes<DT>(la, a.low + (int64_t)li * a.planes * a.r + j, v);
      }
    }
    lds_barrier();
  }
  if (wave >= MG) return;
  // (a wave's row group by its number: unrolled so that ad[] stays in registers)
#pragma unroll
  for (int g = 0; g < MG; ++g) {
    if (wave != g) continue;
    f32x4 v = part[0][g][lane];
#pragma unroll
    for (int q = 1; q < 8; ++q) v += part[q][g][lane];
    const int64_t m = 16 * g + li;
    int todo[1] = {ad[g]};
    for (int cur = next_adapter<1>(todo); cur >= 0; cur = next_adapter<1>(todo)) {
      const bool mine = todo[0] == cur;
      const uint16_t* up = a.up + ((int64_t)cur * a.N + (n0 + li < a.N ? n0 + li : 0)) * a.r;
      f32x4 y = v;
      for (int k0 = 0; k0 < a.cols; k0 += 32) {
        const int kk = k0 + 8 * lg;
        int ku = kk;
        while (ku >= a.r) ku -= a.r;
        uint4 fb = make_uint4(0, 0, 0, 0), fu = make_uint4(0, 0, 0, 0);
        if (kk < a.cols) {
          fb = *reinterpret_cast<const uint4*>(up + ku);
          if (mine) fu = RT > 0 ? *reinterpret_cast<const uint4*>(us + li * ULP + kk)
                                : *reinterpret_cast<const uint4*>(a.low + m * a.planes * a.r + kk);
        }
        y = HT<DT>::mfma16(fb, fu, y);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = mine ? y[i] : v[i];
      todo[0] = mine ? -1 : todo[0];
    }
    const int n = n0 + 4 * lg;
    if (m >= a.rows.M || n >= a.N) continue;  // (N % 8 == 0: whole quadruples)
    if (a.bias) v += *reinterpret_cast<const f32x4*>(a.bias + n);
    if (a.res) {
      if (a.flags & MIMO_EPI_RES_F32) {
        v += *reinterpret_cast<const f32x4*>((const float*)a.res + m * a.ldr + n);
      } else {
        const uint2 h = *reinterpret_cast<const uint2*>((const uint16_t*)a.res + m * a.ldr + n);
        v += (f32x4){HT<DT>::to_f((uint16_t)(h.x & 0xffffu)), HT<DT>::to_f((uint16_t)(h.x >> 16)), HT<DT>::to_f((uint16_t)(h.y & 0xffffu)),
                     HT<DT>::to_f((uint16_t)(h.y >> 16))};
      }
    }
    if (a.flags & MIMO_EPI_OUT_F32) *reinterpret_cast<f32x4*>((float*)a.out + m * a.ldo + n) = v;
    else *reinterpret_cast<uint2*>((uint16_t*)a.out + m * a.ldo + n) = make_uint2(pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]));
  }
}

// ---- host side --------------------------------------------------------------------------------------------------------------
template <int DT>
int launch_low(const LowArgs& a, hipStream_t st) {
  // up to 1024 rows with an index each: a matrix tile would run once per adapter in it, a block per row reads what the row needs.  The
  // order of the rows is not known here: the rule keeps the worst one in bounds and pays for it where requests lie in runs.  Whole call,
  // N = K = 1280, 1024 rows, by rows | by tiles, us:
  //            64 adapters in turn    8 in turn     8 in runs    64 in runs
  //   r = 16       47 |  97            32 | 40       27 | 22       29 | 24
  //   r = 64       90 | 164            59 | 60       49 | 24       56 | 30
  //   r = 128     150 | 356            98 | 115      79 | 30       92 | 44
  // (512 rows alike; 128 rows of 64 adapters in runs 36 | 58, 70 | 93, 116 | 186)
  if (a.rows.rpi == 1 && a.rows.M <= 1024 && a.rows.n > 1) {
    hipLaunchKernelGGL((adapter_low_row_kernel<DT>), dim3((unsigned)a.rows.M), dim3(256), 0, st, a);
    MIMO_LAUNCH_CHECK();
    return MIMO_OK;
  }
  const int rt = (a.r + 15) / 16;
  const int64_t m32 = (a.rows.M + 31) / 32;
  // one wave per 32 rows would leave SIMDs empty (whole call, N = K = 640, r = 16: 30.5 us split, 33.1 not, at M = 16384; 69.7 and 67.7
  // at M = 49152)
  const bool ksplit = m32 < 4 * (int64_t)cu_count();
  const int64_t nwg = ksplit ? m32 : (m32 + 3) / 4;
  if (nwg > 0x7fffffff) return MIMO_EINVAL;
#define LOW(RT)                                                                                                                  \
  do {                                                                                                                           \
    if (ksplit) hipLaunchKernelGGL((adapter_low_kernel<DT, RT, true>), dim3((unsigned)nwg), dim3(64 * low_waves(RT, true)), 0, st, a); \
    else hipLaunchKernelGGL((adapter_low_kernel<DT, RT, false>), dim3((unsigned)nwg), dim3(256), 0, st, a);                      \
  } while (0)
  if (rt == 1) LOW(1);
  else if (rt == 2) LOW(2);
  else if (rt <= 4) LOW(4);
  else LOW(8);
#undef LOW
  MIMO_LAUNCH_CHECK();
  return MIMO_OK;
}

template <int DT, int NR>
int launch_tiles(GemmArgs& g, hipStream_t st) {
  // the tile choice of mimo_gemm (gemm_conv.hip launch_nr), without split-K and persistent blocks
  const int cus = cu_count();
  const int64_t m256 = (g.M + 255) / 256;
  const int tn_s = (g.N + 32 * NR - 1) / (32 * NR), tn_xl = (g.N + 64 * NR - 1) / (64 * NR);
  if (g.N > 32 * NR && m256 * tn_xl >= 160) {
    g.tiles_n = tn_xl;
    auto cost = [&](int bm) { return ((((g.M + bm - 1) / bm) * tn_xl + cus - 1) / cus) * (int64_t)(bm + 24); };
    int bm = 256;
    if (cost(192) < cost(bm)) bm = 192;
    if (cost(128) < cost(bm)) bm = 128;
    const int64_t nwg = ((g.M + bm - 1) / bm) * tn_xl;
    if (nwg > 0x7fffffff) return MIMO_EINVAL;
    if (bm == 256) {
      hipLaunchKernelGGL((gemm_kernel<DT, NR, 0, 2, 4, 2, 8, 3>), dim3((unsigned)nwg), dim3(512), 0, st, g);
    } else if (bm == 192) {
      hipLaunchKernelGGL((gemm_kernel<DT, NR, 0, 2, 4, 2, 6, 3>), dim3((unsigned)nwg), dim3(512), 0, st, g);
    } else {
      hipLaunchKernelGGL((gemm_kernel<DT, NR, 0, 2, 4, 2, 4, 3>), dim3((unsigned)nwg), dim3(512), 0, st, g);
    }
  } else {
    g.tiles_n = tn_s;
    const int64_t nwg = ((g.M + 127) / 128) * tn_s;
    if (nwg > 0x3fffffff) return MIMO_EINVAL;
    if (nwg <= cus) {
      // (128-column tiles: three ring slots of 64 x 128 leave room for a second block per CU)
      g.tiles_n = (g.N + 127) / 128;
      const int64_t nwg64 = ((g.M + 63) / 64) * g.tiles_n;
      hipLaunchKernelGGL((gemm_kernel<DT, 4, 0, 2, 2, 3, 2, 3>), dim3((unsigned)nwg64), dim3(256), 0, st, g);
    } else {
      hipLaunchKernelGGL((gemm_kernel<DT, NR, 0, 2, 2, 2, 4, 3>), dim3((unsigned)nwg), dim3(256), 0, st, g);
    }
  }
  MIMO_LAUNCH_CHECK();
  return MIMO_OK;
}

template <int DT>
int launch_gemm(GemmArgs g, hipStream_t st) {
  // operands are addressed with 32-bit byte offsets: more rows than that go in several launches
  const int64_t M = g.M, wide = g.lda > g.ad_ld ? g.lda : g.ad_ld, most = (0x7fffffffLL / (2 * wide) - 1) / 256 * 256;
  const bool of32 = g.flags & MIMO_EPI_OUT_F32, rf32 = g.flags & MIMO_EPI_RES_F32;
  for (int64_t r0 = 0; r0 < M; r0 += most) {
    GemmArgs c = g;
    c.M = M - r0 < most ? M - r0 : most;
    c.A = g.A + r0 * g.lda;
    c.out = (char*)g.out + r0 * g.ldo * (of32 ? 4 : 2);
    if (g.res) c.res = (const char*)g.res + r0 * g.ldr * (rf32 ? 4 : 2);
    c.ad_row0 = r0;
    c.ad_low = g.ad_low + r0 * g.ad_ld;
    c.a_bytes = (unsigned)(((c.M - 1) * c.lda + c.K) * 2);
    const int64_t tn8 = (c.N + 255) / 256, nt8 = ((c.M + 255) / 256) * tn8;
    int rc;
    // (256 x 256 tiles once they fill three quarters of the chip: the whole call 104 us against 112 with the other tiles at 245 of them,
    // M = 12321, N = K = 1280, r = 64, fp32 out, sixteen requests, and 80 against 90 with one; 44.8 against 39.3 at 160, M = 8192, r = 16)
    if ((c.K % 64) == 0 && tn8 * 256 - c.N <= c.N / 12 && 4 * nt8 >= 3 * (int64_t)cu_count() && nt8 <= 0x7fffffff) {
      c.tiles_n = (int)tn8;
      c.ntiles = (unsigned)G8_GM;
      hipLaunchKernelGGL((gemm8_kernel<DT, 3>), dim3((unsigned)nt8), dim3(512), 0, st, c);
      const hipError_t e = hipGetLastError();
      rc = e == hipSuccess ? MIMO_OK : (int)e;
    } else {
      rc = c.N % 160 == 0 ? launch_tiles<DT, 5>(c, st) : launch_tiles<DT, 4>(c, st);
    }
    if (rc) return rc;
  }
  return MIMO_OK;
}

// checks shared by both entries
int check(const mimo_adapter_params* p, int64_t M, int N, int K) {
  if (!p || M <= 0 || M >= 0x7fffffffLL || N <= 0 || K <= 0 || (N & 7) || (K & 7) || (int64_t)N * K >= 0x40000000LL ||
      N >= 0x100000 || K >= 0x100000)
    return MIMO_EINVAL;
  if (!p->down || !p->up || !p->index || p->count <= 0 || p->rank <= 0 || p->rank > 128 || (p->rank & 7) || p->rows_per_index <= 0)
    return MIMO_EINVAL;
  if (p->count > 65535 || !aligned16(p->down) || !aligned16(p->up) || (reinterpret_cast<uintptr_t>(p->index) & 3u)) return MIMO_EINVAL;
  return MIMO_OK;
}

Rows rows_of(const mimo_adapter_params* p, int64_t M) {
  return Rows{p->index, M, (unsigned)(p->rows_per_index < 0x7fffffff ? p->rows_per_index : 0x7fffffff), p->count};
}

GemmArgs gemm_args(const void* A, int64_t lda, const void* W, void* out, int64_t ldo, int64_t M, int N, int K, const Rows& rows,
                   const uint16_t* low, int ld, int cols, const uint16_t* up, int rank) {
  GemmArgs g{};
  g.A = (const uint16_t*)A; g.W = (const uint16_t*)W; g.out = out;
  g.lda = lda; g.ldw = K; g.ldo = ldo; g.M = M; g.N = N; g.K = K; g.out_scale = 1.f;
  g.rows_per_img = 1; g.ldib = N; g.ln_rows_per_frame = 1; g.ln_pe_frames = 1;
  g.nkt = (K + BK - 1) / BK;
  g.w_bytes = (unsigned)((int64_t)N * K * 2);
  g.flags = F_STAGGER;
  g.ad_index = rows.index; g.ad_rpi = rows.rpi; g.ad_n = rows.n;
  g.ad_low = low; g.ad_up = up; g.ad_rank = rank; g.ad_cols = cols; g.ad_ld = ld;
  return g;
}

// Up to 64 rows: the skinny kernel (whole call, N = K = 1280, r = 16: 21.3 us for 8 rows and for 64, by the tiles 23.9 and 30.0; N = K =
// 320, 64 rows: 21.2 against 21.7); u inside it for up to four rows, whose adapters it takes one after another (four rows 18.7 us against
// 21.4 with a launch for u; eight rows of different adapters: one kernel of 20.1 us, two of 14.5 together).
template <int DT>
int launch_skinny(const GemmArgs& g, const LowArgs& la, hipStream_t st) {
  SkinnyArgs a{g.A, g.W, la.down, g.ad_up, la.scale, g.bias, g.res, g.out, la.low, g.lda, g.ldo, g.ldr, la.rows,
               g.N, g.K, la.r, la.planes, g.ad_cols, g.flags};
  const dim3 grid((unsigned)((g.N + 15) / 16));
  const int rt = (la.r + 15) / 16, mg = (int)((g.M + 15) / 16);
  if (g.M <= 4 && rt <= 4) {
    if (rt == 1) hipLaunchKernelGGL((adapter_skinny_kernel<DT, 1, 1>), grid, dim3(512), 0, st, a);
    else if (rt == 2) hipLaunchKernelGGL((adapter_skinny_kernel<DT, 1, 2>), grid, dim3(512), 0, st, a);
    else hipLaunchKernelGGL((adapter_skinny_kernel<DT, 1, 4>), grid, dim3(512), 0, st, a);
    MIMO_LAUNCH_CHECK();
    return MIMO_OK;
  }
  if (const int rc = launch_low<DT>(la, st)) return rc;
  if (mg == 1) hipLaunchKernelGGL((adapter_skinny_kernel<DT, 1, 0>), grid, dim3(512), 0, st, a);
  else if (mg == 2) hipLaunchKernelGGL((adapter_skinny_kernel<DT, 2, 0>), grid, dim3(512), 0, st, a);
  else hipLaunchKernelGGL((adapter_skinny_kernel<DT, 4, 0>), grid, dim3(512), 0, st, a);
  MIMO_LAUNCH_CHECK();
  return MIMO_OK;
}

template <int DT>
int forward(const GemmArgs& g, const LowArgs& la, hipStream_t st) {
  if (g.M <= 64) return launch_skinny<DT>(g, la, st);
  if (const int rc = launch_low<DT>(la, st)) return rc;
  return launch_gemm<DT>(g, st);
}

// workspace of the backward, in bytes: t [M, planes r] | up^T | down^T | parts of ddown | parts of dup
struct BackwardPlan {
  int parts;
  size_t t, upt, downt, p0, p1, total;
};
BackwardPlan backward_plan(int dtype, const mimo_adapter_params* p, int64_t M, int N, int K) {
  BackwardPlan b{};
  const int64_t n = p->count, r = p->rank;
  const int64_t blocks = n * ((N + 127) / 128 + (K + 127) / 128), tiles = (M + 63) / 64;
  int64_t parts = (3 * (int64_t)cu_count() + blocks - 1) / blocks;  // three blocks per CU; a part keeps at least four row tiles
  if (parts > tiles / 4) parts = tiles / 4;
  if (parts > 256) parts = 256;
  b.parts = parts < 1 ? 1 : (int)parts;
  auto up16 = [](size_t x) { return (x + 15) / 16 * 16; };
  b.t = up16((size_t)M * planes_of(dtype) * r * 2);
  b.upt = up16((size_t)n * r * N * 2);
  b.downt = up16((size_t)n * r * K * 2);
  b.p0 = up16((size_t)b.parts * n * r * K * 4);
  b.p1 = up16((size_t)b.parts * n * r * N * 4);
  b.total = b.t + b.upt + b.downt + b.p0 + b.p1;
  return b;
}

template <int DT>
int backward(const void* dY, int64_t ldy, const void* A, int64_t lda, const void* Wt, void* dA, int64_t ldda, int64_t M, int N, int K,
             const mimo_adapter_params* p, const void* low, float* ddown, float* dup, char* ws, hipStream_t st) {
  const BackwardPlan b = backward_plan(DT, p, M, N, K);
  const int n = p->count, r = p->rank;
  uint16_t* t = (uint16_t*)ws;
  uint16_t* upt = (uint16_t*)(ws + b.t);
  uint16_t* downt = (uint16_t*)(ws + b.t + b.upt);
  float* p0 = (float*)(ws + b.t + b.upt + b.downt);
  float* p1 = (float*)((char*)p0 + b.p0);
  const Rows rows = rows_of(p, M);
  TransposeArgs ta{{(const uint16_t*)p->up, (const uint16_t*)p->down}, {upt, downt}, {N, r}, {r, K}};
  const int tiles = ((N > K ? N : K) + 31) / 32 * ((r + 31) / 32);
  hipLaunchKernelGGL(adapter_transpose_kernel, dim3((unsigned)tiles, (unsigned)n, 2u), dim3(256), 0, st, ta);
  MIMO_LAUNCH_CHECK();
  constexpr int NP = planes_of(DT);
  constexpr float up2 = DT == MIMO_F16 ? T_SCALE : 1.f;
  const LowArgs la{(const uint16_t*)dY, upt, p->scale, t, ldy, rows, N, r, NP, up2};
  if (const int rc = launch_low<DT>(la, st)) return rc;
  if (dA) {
    GemmArgs g = gemm_args(dY, ldy, Wt, dA, ldda, M, K, N, rows, t, NP * r, r, downt, r);
    if (const int rc = launch_gemm<DT>(g, st)) return rc;
  }
  OuterArgs oa{{(const uint16_t*)A, (const uint16_t*)dY}, {t, (const uint16_t*)low}, {p0, p1}, {lda, ldy}, {K, N}, {1.f / up2, 1.f}, rows, r,
               (K + 127) / 128, fast_div(rows.rpi), fast_div((uint32_t)(NP * r / 8))};
  const dim3 grid((unsigned)((K + 127) / 128 + (N + 127) / 128), (unsigned)n, (unsigned)b.parts);
  const int rt = (r + 15) / 16;
  if (rt == 1) hipLaunchKernelGGL((adapter_outer_kernel<DT, 1>), grid, dim3(256), 0, st, oa);
  else if (rt == 2) hipLaunchKernelGGL((adapter_outer_kernel<DT, 2>), grid, dim3(256), 0, st, oa);
  else if (rt <= 4) hipLaunchKernelGGL((adapter_outer_kernel<DT, 4>), grid, dim3(256), 0, st, oa);
  else hipLaunchKernelGGL((adapter_outer_kernel<DT, 8>), grid, dim3(256), 0, st, oa);
  MIMO_LAUNCH_CHECK();
  const int64_t total = (int64_t)n * r * (N + K), nwg = (total / 4 + 31) / 32;
  if (nwg > 0x7fffffff) return MIMO_EINVAL;
  hipLaunchKernelGGL(adapter_join_kernel, dim3((unsigned)nwg), dim3(256), 0, st, p0, p1, ddown, dup, n, r, K, N,
                     b.parts);
  MIMO_LAUNCH_CHECK();
  return MIMO_OK;
}

}  // namespace

extern "C" int mimo_adapter_gemm(int dtype, const void* A, int64_t lda, const void* W, void* out, int64_t ldo, int64_t M, int N, int K,
                                 const float* bias, const void* residual, int64_t ldr, unsigned flags, const mimo_adapter_params* p,
                                 void* low, int low_split, void* stream) {
  if (const int rc = check(p, M, N, K)) return rc;
  if (!A || !W || !out || !low || (lda & 7) || (ldo & 3) || (residual && (ldr & 3)) || !aligned16(A) || !aligned16(W) || !aligned16(out) ||
      !aligned16(low) || lda < 0 || lda > 0x100000 || ldo < 0 || ldo > 0x100000 || (residual && (ldr < 0 || ldr > 0x100000)))
    return MIMO_EINVAL;
  if (flags & ~(MIMO_EPI_OUT_F32 | MIMO_EPI_RES_F32)) return MIMO_EINVAL;
  const bool of32 = flags & MIMO_EPI_OUT_F32;
  if (of32 && !low_split) return MIMO_EINVAL;
  const Rows rows = rows_of(p, M);
  if (dtype != MIMO_F16 && dtype != MIMO_BF16) return MIMO_EDTYPE;
  const int planes = low_split ? planes_of(dtype) : 1;
  GemmArgs g = gemm_args(A, lda, W, out, ldo, M, N, K, rows, (const uint16_t*)low, planes * p->rank, of32 ? planes * p->rank : p->rank,
                         (const uint16_t*)p->up, p->rank);
  g.bias = bias; g.res = residual; g.ldr = ldr;
  g.flags |= flags;
  const LowArgs la{(const uint16_t*)A, (const uint16_t*)p->down, p->scale, (uint16_t*)low, lda, rows, K, p->rank, planes, 1.f};
  return dtype == MIMO_F16 ? forward<MIMO_F16>(g, la, (hipStream_t)stream) : forward<MIMO_BF16>(g, la, (hipStream_t)stream);
}

extern "C" size_t mimo_adapter_gemm_backward_workspace(int dtype, const mimo_adapter_params* p, int64_t M, int N, int K) {
  return check(p, M, N, K) == MIMO_OK ? backward_plan(dtype, p, M, N, K).total : 0;
}

extern "C" int mimo_adapter_gemm_backward(int dtype, const void* dY, int64_t ldy, const void* A, int64_t lda, const void* Wt, void* dA,
                                          int64_t ldda, int64_t M, int N, int K, const mimo_adapter_params* p, const void* low,
                                          float* ddown, float* dup, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int rc = check(p, M, N, K)) return rc;
  if (!dY || !A || !low || !ddown || !dup || !workspace || (dA && !Wt) || (ldy & 7) || (lda & 7) || (ldda & 3) || lda < 0 || ldy < 0 || ldy > 0x100000 ||
      ldda < 0 || ldda > 0x100000 ||
      !aligned16(dY) || !aligned16(A) || !aligned16(Wt) || !aligned16(dA) || !aligned16(low) || !aligned16(ddown) || !aligned16(dup) ||
      !aligned16(workspace) || workspace_bytes < backward_plan(dtype, p, M, N, K).total)
    return MIMO_EINVAL;
  if (dtype == MIMO_F16)
    return backward<MIMO_F16>(dY, ldy, A, lda, Wt, dA, ldda, M, N, K, p, low, ddown, dup, (char*)workspace, (hipStream_t)stream);
  if (dtype == MIMO_BF16)
    return backward<MIMO_BF16>(dY, ldy, A, lda, Wt, dA, ldda, M, N, K, p, low, ddown, dup, (char*)workspace, (hipStream_t)stream);
  return MIMO_EDTYPE;
}
