// cross_attention.hip.h — what the forward and the backward kernels of the cross attention share: arguments, the flat query
// rows, the masked staging of key / value rows, transposed LDS fragments (gfx950, MFMA 32x32x16).
//
// Work is laid out per (encoder row e, key head g).  The queries that see these keys are the images [e G, (e + 1) G), their Nq
// tokens and the hg query heads of the key head: R = G Nq hg FLAT ROWS, f = (image, token, head) with the head fastest.  A wave
// takes 32 of them as the 32 columns of a matrix tile, so 24 single-token frames or 8 grouped heads of one token fill a tile
// as well as 32 neighbouring tokens do.
#pragma once
#include "common.hip.h"

namespace mimo_xattn {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct Args {
  const uint16_t *q, *k, *v;
  const uint16_t *o, *dout;      // backward: the forward's output and its gradient
  const float* lse_in;           // backward
  uint16_t *out, *dk, *dv;       // out: the forward's output, or dq
  float *lse, *delta;            // [B, heads, Nq]
  float* ws;                     // partial results of a split launch
  int* tops;                     // backward, fp16: [Be kvh][slots] exponents of bounds of |dS|, one per wave of dq, for dk / dv
  const int* kv_len;             // [Be] or null
  const uint8_t* mask;           // [Be, Nk] or null
  int64_t sqb, sqr, skb, skr, svb, svr, sob, sor, sdb, sdr, smb;  // element strides: batch, row (o / dout: sob.., sdb..)
  int Be, G, Nq, Nk, kvh, hg, d, R;
  FastDiv by_hg, by_nq, by_dc;   // query heads per key head, tokens, 16-byte chunks of a head
  float c;                       // scale * log2(e): scores leave the matrix unit unscaled
  float scale, lag;
  int nb;                        // blocks per (e, g)
  int slots;                     // waves of dq per (e, g)
  int nsplit;                    // parts the keys (forward) or the flat rows (dk / dv) are cut into; dq takes all keys in one
};

// (image, token, head) of a flat row
__device__ __forceinline__ void flat_row(const Args& a, int f, int& img, int& qi, int& hh) {
  const uint32_t t = div_fast((uint32_t)f, a.by_hg);
  hh = f - (int)t * a.hg;
  img = (int)div_fast(t, a.by_nq);
  qi = (int)t - img * a.Nq;
}

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }  // arguments <= ~0: flushing is fine

__device__ __forceinline__ int valid_len(const Args& a, int e) {
  if (!a.kv_len) return a.Nk;
  const int n = a.kv_len[e];
  return n < 0 ? 0 : (n > a.Nk ? a.Nk : n);
}
__device__ __forceinline__ bool key_valid(const Args& a, int e, int len, int key) {
  return key < len && (!a.mask || a.mask[(int64_t)e * a.smb + key]);
}

// A operand of a 32x32x16 MFMA from a row-major LDS tile with rows = the contraction index: lane (h2, i = lane & 31) gets
// column c0 + i of rows {r0 + 4 h2 + 0..3, r0 + 8 + 4 h2 + 0..3} — the k-slot order in which a 32x32 accumulator tile holds its
// 16 consecutive rows, so that packed accumulators are the B operand without a lane exchange.  Two hardware-transposed reads:
// inside a 16-lane group lane m points at row (m >> 2), columns 4 (m & 3).., lane i receives column i of the four rows.
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
__device__ __forceinline__ uint4 read_tr(const uint16_t* tile, int pitch, int r0, int c0, int lane) {
  const int m = lane & 15, cg = (lane >> 4) & 1, h2 = lane >> 5;
  const uint16_t* p = tile + (r0 + 4 * h2 + (m >> 2)) * pitch + c0 + 16 * cg + 4 * (m & 3);
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)p);
  const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(p + 8 * pitch));
  const uint2 lo = __builtin_bit_cast(uint2, a), hi = __builtin_bit_cast(uint2, b);
  return make_uint4(lo.x, lo.y, hi.x, hi.y);
}

// eight packed accumulator rows [8 u, 8 u + 8) of a 32x32 tile = the k-step u of the product that contracts over its rows
template <int DT>
__device__ __forceinline__ uint4 pack_k(const f32x16& s, int u) {
  return make_uint4(pack2<DT>(s[8 * u], s[8 * u + 1]), pack2<DT>(s[8 * u + 2], s[8 * u + 3]),
                    pack2<DT>(s[8 * u + 4], s[8 * u + 5]), pack2<DT>(s[8 * u + 6], s[8 * u + 7]));
}

// Where the 32 flat rows of tile t go in a contiguous [B, Nq, heads d] tensor and in a [B, heads, Nq] table: uniform bases plus
// 32-bit lane offsets for buffer stores, out of range for rows that do not exist.  No store is behind a branch: the loop knows how
// many follow the next tile's loads and waits for those loads alone, not for the stores' acknowledgement.
struct RowPlace {
  __amdgpu_buffer_rsrc_t out, table;
  unsigned row, stat;
};
__device__ __forceinline__ RowPlace row_place(const Args& a, int e, int g, int t, int li, uint16_t* out, float* table) {
  RowPlace p;
  const int f = 32 * t + li;
  int img, qi, hh;
  flat_row(a, f < a.R ? f : a.R - 1, img, qi, hh);
  const uint32_t tq0 = div_fast((uint32_t)(32 * t), a.by_hg), img0 = div_fast(tq0, a.by_nq);
  const int heads = a.kvh * a.hg, head = g * a.hg + hh, C = heads * a.d;
  p.out = __builtin_amdgcn_make_buffer_rsrc(out + ((int64_t)e * a.G * a.Nq + tq0) * C, 0, 0x7fffffff, 0x00020000);
  p.table = __builtin_amdgcn_make_buffer_rsrc(table + ((int64_t)e * a.G + img0) * heads * a.Nq, 0, table ? 0x7fffffff : 0, 0x00020000);
  p.row = f < a.R ? (unsigned)((img * a.Nq + qi - (int)tq0) * C + head * a.d) * 2u : 0xF0000000u;
  p.stat = f < a.R ? (unsigned)(((img - (int)img0) * heads + head) * a.Nq + qi) * 4u : 0xF0000000u;
  return p;
}

// stores 32 channels (tile dt) of the flat rows a 32x32 accumulator tile holds as columns: the two lane halves exchange
// quadruples so that a lane writes 16 bytes.
template <int DT>
__device__ __forceinline__ void store_tile(const f32x16& o, float f, const RowPlace& p, int dt, int d, int h2) {
  typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int c = 0; c < 4; c += 2) {
    const auto x = __builtin_amdgcn_permlane32_swap(pack2<DT>(o[4 * c] * f, o[4 * c + 1] * f),
                                                    pack2<DT>(o[4 * c + 4] * f, o[4 * c + 5] * f), false, false);
    const auto y = __builtin_amdgcn_permlane32_swap(pack2<DT>(o[4 * c + 2] * f, o[4 * c + 3] * f),
                                                    pack2<DT>(o[4 * c + 6] * f, o[4 * c + 7] * f), false, false);
    const int d0 = 32 * dt + 8 * c + 8 * h2;
    const u32x4 v = {x[0], y[0], x[1], y[1]};
    __builtin_amdgcn_raw_buffer_store_b128(v, p.out, d0 < d ? p.row + 2u * (unsigned)d0 : 0xF0000000u, 0, 0);
  }
}

// fragments of one row: lane (h2, .) holds channels 16 s + 8 h2 .. + 8.  Channels >= d repeat channel 0 (the partner operand
// is zero there); rows that do not exist are the caller's to drop.
template <int KS>
__device__ __forceinline__ void load_row(uint4 (&f)[KS], const uint16_t* p, int d, int h2) {
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int kk = 16 * s + 8 * h2;
    f[s] = *reinterpret_cast<const uint4*>(p + (kk < d ? kk : 0));
  }
}

// waits for requested fragments HERE.  Used first inside a loop that keeps other requests on their way, they would be waited for
// in every round of it, and the younger requests with them.
template <int KS>
__device__ __forceinline__ void settle(uint4 (&f)[KS]) {
#pragma unroll
  for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(f[s].x), "+v"(f[s].y), "+v"(f[s].z), "+v"(f[s].w));
}

// lanes per row of 16-byte chunks: a power of two, so that a thread keeps its columns and walks rows at a fixed distance; at most
// eight (a line of 128 bytes), which take wider rows in several chunks each: a row's address is made once for all of them
constexpr int lanes_of(int ks) { return ks <= 2 ? 4 : 8; }
constexpr int chunks_of(int ks) { return (2 * ks + lanes_of(ks) - 1) / lanes_of(ks); }

// the larger magnitudes of two running fp16 maxima (bits without sign: they order like integers, NaN on top) and of eight halfs
__device__ __forceinline__ uint32_t top_of(uint32_t top, uint4 y) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  u16x2 m = __builtin_bit_cast(u16x2, top);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, (i == 0 ? y.x : i == 1 ? y.y : i == 2 ? y.z : y.w) & 0x7fff7fffu));
  return __builtin_bit_cast(uint32_t, m);
}

// Key and value rows [key0, key0 + N) of (e, g) on their way into row-major LDS tiles of pitch 16 KS + 8 halfs (an odd number of
// 16-byte units: a 16-lane group of b128 row reads covers all banks).  issue() requests the rows, commit() writes them: between
// the two a block computes on other rows.  Only keys below len are read; what the mask drops, rows behind len and channels
// >= d are ZERO in LDS whatever memory holds there (NaN included), and bias[i] = 0 or -inf is added to their scores.
// ones: V's channel d, which pads the last 32-channel tile, is 1 — the product with P then also leaves the sum of P in that row.
// TOP (fp16): top collects the largest |v| of what is written, as bits, two maxima in one word.
template <int KS, int THREADS, int N>
struct Stager {
  static constexpr int P = 16 * KS + 8, LPR = lanes_of(KS), CH = chunks_of(KS), RP = THREADS / LPR, NC = (N + RP - 1) / RP;
  uint4 kr[NC][CH], vr[NC][CH];
  uint8_t keep;  // the mask's byte of key key0 + lane
  int left;      // keys of this piece
  uint32_t top = 0u;
  const uint16_t *kb, *vb;
  __device__ __forceinline__ void open(const Args& a, int e, int g) {
    kb = a.k + (int64_t)e * a.skb + (int64_t)g * a.d;
    vb = a.v + (int64_t)e * a.svb + (int64_t)g * a.d;
  }
  // (no select between the requests: keys behind the last one repeat it)
  __device__ __forceinline__ void issue(const Args& a, int e, int len, int key0, int tid) {
    asm volatile("" : "+v"(tid));  // addresses are made anew for every piece: kept over the products they would cost registers
    const int row0 = tid / LPR, cc = (tid & (LPR - 1)) * 8;
    left = len - key0;  // > 0
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int key = key0 + min(row0 + i * RP, left - 1);
      const uint16_t *kp = kb + (int64_t)key * a.skr + cc, *vp = vb + (int64_t)key * a.svr + cc;
#pragma unroll
      for (int c = 0; c < CH; ++c)
        if (cc + 8 * LPR * c < a.d) {
          kr[i][c] = *reinterpret_cast<const uint4*>(kp + 8 * LPR * c);
          vr[i][c] = *reinterpret_cast<const uint4*>(vp + 8 * LPR * c);
        }
    }
    static_assert(N <= 64, "a lane per key of the mask");
    keep = 1;
    if (a.mask) keep = a.mask[(int64_t)e * a.smb + key0 + min(tid & 63, left - 1)];
  }
  template <int DT, bool TOP = false>
  __device__ __forceinline__ void commit(const Args& a, uint16_t* ks, uint16_t* vs, float* bias, bool ones, int tid) {
    asm volatile("" : "+v"(tid));
    const int row0 = tid / LPR, cc = (tid & (LPR - 1)) * 8;
    const bool mine = (tid & 63) < left && keep != 0;
    const unsigned long long live = __builtin_amdgcn_ballot_w64(mine);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int row = row0 + i * RP;
      const bool alive = (live >> (row & 63)) & 1;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int col = cc + 8 * LPR * c;
        if (col < 16 * KS && (N % RP == 0 || row < N)) {
          const bool ok = alive && col < a.d;
          uint4 x = ok ? kr[i][c] : make_uint4(0, 0, 0, 0), y = ok ? vr[i][c] : make_uint4(0, 0, 0, 0);
          if constexpr (TOP) top = top_of(top, y);
          if (ones && col == a.d) y.x = HT<DT>::from_f(1.f);
          *reinterpret_cast<uint4*>(ks + row * P + col) = x;
          *reinterpret_cast<uint4*>(vs + row * P + col) = y;
        }
      }
    }
    if (tid < N) {
      bias[tid] = mine ? 0.f : -INFINITY;
      if (ones && a.d == 16 * KS) vs[tid * P + a.d] = HT<DT>::from_f(1.f);
    }
  }
};

// all keys of (e, g), 96 at a time on their way; the thread's top (0 without TOP)
template <int DT, int KS, int THREADS, bool TOP = false>
__device__ __forceinline__ uint32_t stage_all(const Args& a, int e, int g, int len, uint16_t* ks, uint16_t* vs, float* bias, bool ones, int tid) {
  constexpr int P = 16 * KS + 8;
  uint32_t top = 0u;
  for (int k0 = 0; k0 < len; k0 += 96) {
    Stager<KS, THREADS, 32> s[3];
#pragma unroll
    for (int u = 0; u < 3; ++u)
      if (k0 + 32 * u < len) {
        s[u].open(a, e, g);
        s[u].issue(a, e, len, k0 + 32 * u, tid);
      }
#pragma unroll
    for (int u = 0; u < 3; ++u)
      if (k0 + 32 * u < len) {
        s[u].top = top;
        s[u].template commit<DT, TOP>(a, ks + (k0 + 32 * u) * P, vs + (k0 + 32 * u) * P, bias + k0 + 32 * u, ones, tid);
        top = s[u].top;
      }
  }
  return top;
}

// bytes of LDS that n staged keys take (+ the transposed reads of the last row's last tile, which run up to 16 halfs past it)
constexpr int kv_lds(int ks, int n) { return 2 * n * (16 * ks + 8) * 2 + n * 4 + 64; }

inline int cu_count() {
  static const int cus = [] {
    int dev = 0, n = 0;
    if (hipGetDevice(&dev) != hipSuccess ||
        hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
    return n;
  }();
  return cus;
}

// the padded head widths that have kernels: 16 KS halfs, KS = 2 3 4 5 6 8 10
inline int k_steps(int d) { return d <= 32 ? 2 : d <= 48 ? 3 : d <= 64 ? 4 : d <= 80 ? 5 : d <= 96 ? 6 : d <= 128 ? 8 : 10; }

#define MIMO_XATTN_DISPATCH(ks, CALL) \
  switch (ks) {                       \
    case 2: CALL(2); break;           \
    case 3: CALL(3); break;           \
    case 4: CALL(4); break;           \
    case 5: CALL(5); break;           \
    case 6: CALL(6); break;           \
    case 8: CALL(8); break;           \
    default: CALL(10); break;         \
  }

// fills the geometry; MIMO_OK or an error.  Strides are those of the header's mimo_cross_attention_params.
int fill(Args& a, const mimo_cross_attention_params* p);

}  // namespace mimo_xattn
