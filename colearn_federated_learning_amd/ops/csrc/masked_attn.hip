// Self-attention with document masks, causal and prefix masks, capped scores
// and linear distance biases, for any length; forward and backward, bf16 or
// fp16 operands, head sizes up to 128, shared key heads.
//
//   z_ij = scale q_i.k_j;  z = cap tanh(z / cap);  z -= slope_h |i - j|
//   (i, j) attended:  doc_i == doc_j >= 0  and  (not causal or j <= i or
//                     j < prefix)
//   p = softmax of z over the attended j (all 0 if there is none),  o = p v
//   D_i = go_i.o_i;  dp = go v^T;  dz = p (dp - D) (1 - tanh^2)
//   dq = scale dz k,  dk = scale dz^T q,  dv = p^T go
//
// All three kernels have one shape.  A wave owns 32 tokens (queries in the
// forward and dq kernels, keys in the dk/dv kernel) whose operands stay in
// registers, and tiles of 64 tokens of the other side stream through LDS,
// double-buffered: the next tile's loads are issued before a tile is worked
// on and land in the other buffer after it.  Products are 32x32x16 MFMAs with
// the streamed side as the left operand, so that a lane's column of the
// result belongs to one owned token and its 16 registers to streamed tokens:
// the softmax is a reduction over registers plus one exchange between the
// wave's halves, and the rounded probabilities already lie as the right
// operand of the second product.  That operand's k order is
//     slot 8h + j  <->  token 4h + (j & 3) + 8 (j >> 2)       (h: lane / 32)
// instead of the plain one; the left operand, read transposed from the same
// LDS tile (ds_read_b64_tr_b16: four tokens of 16 columns a lane group), uses
// the same order, so nothing moves between lanes.
//
// In fp16 the backward rounds 2^15 p instead of p (the factor leaves dv again
// in fp32): a uniform row of 16K tokens has p = 2^-14, below which fp16 loses
// a bit for every halving.  dz has no such bound and is rounded as it is.
//
// Scores are held in base 2 (scale * log2 e folded in) and every statistic in
// fp32.  Probabilities and dz are rounded to the operands' type for the second
// products; the sums in the denominator are of the unrounded ones.
//
// The mask is summarised per 64 tokens (smallest and largest document, any
// padding).  A workgroup first lists the tiles that it has to visit, each
// marked whole (every pair attended: no test in the loop) or mixed; tiles
// between documents that do not meet cost nothing.  Rows of padding are
// staged as zeros and rows of padding are written as zeros, so that whatever
// a padded token holds reaches no result.
//
// The backward recomputes p from the saved row statistic, in two kernels
// without atomics (dq with D, then dk/dv): 7 products instead of the 5 of a
// single kernel whose dq would be summed by atomics in an order that changes
// from run to run.

#include "elem.h"
#include "encoder_api.h"

namespace colearn {

namespace {

constexpr int kTile = kAttnTile;   // streamed tokens a tile
constexpr int kOwn = 128;          // owned tokens a workgroup, 32 a wave
constexpr int kList = 1024;        // tiles listed at a time
constexpr float kLog2e = 1.4426950408889634f;

typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(8))) float f32x8;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

template <typename T>
DEV_INLINE f32x16 mfma(s16x8 a, s16x8 b, f32x16 c);
template <>
DEV_INLINE f32x16 mfma<bf16>(s16x8 a, s16x8 b, f32x16 c) {
  typedef __attribute__((ext_vector_type(8))) __bf16 V;
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(
      __builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
}
template <>
DEV_INLINE f32x16 mfma<f16>(s16x8 a, s16x8 b, f32x16 c) {
  typedef __attribute__((ext_vector_type(8))) _Float16 V;
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(
      __builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
}

// registers 8k .. 8k+7 of a result, rounded to T
template <typename T>
DEV_INLINE s16x8 round8(const f32x16& x, int k) {
  typedef __attribute__((ext_vector_type(8))) typename Bits16<T>::hw V;
  f32x8 f;
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = x[8 * k + j];
  return __builtin_bit_cast(s16x8, __builtin_convertvector(f, V));
}

// what a probability is multiplied with before it is rounded, in the backward
template <typename T>
constexpr float kLift = 1.f;
template <>
constexpr float kLift<f16> = 32768.f;

DEV_INLINE float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// tanh from one exponential and one reciprocal; off by about 1e-7, far below
// the rounding of the products around it
DEV_INLINE float fast_tanh(float x) {
  const float e = fast_exp2(x * (2.f * kLog2e));
  return 1.f - 2.f * __builtin_amdgcn_rcpf(e + 1.f);
}

// the other half's value (lane ^ 32)
DEV_INLINE float other_half(float x) { return __shfl_xor(x, 32); }

// A tile of kTile rows of DP 16-bit values.  16-byte slots are permuted
// within a row so that neither read below hits a bank twice: eight
// consecutive rows of a slot (row operand) lie over all slots of 128 bytes,
// and so do four consecutive rows of two slots (transposed operand).
template <int DP>
struct Tile {
  static constexpr int kSlots = DP / 8;
  static constexpr int kPer = kTile * kSlots / 256;  // slots a thread
  static constexpr int kBytes = kTile * DP * 2;

  DEV_INLINE static int at(int row, int slot) {
    const int f = DP == 32 ? ((row & 2) | ((row >> 2) & 1))
                           : (((row & 3) << 1) | ((row >> 2) & 1));
    return row * (DP * 2) + ((slot ^ f) << 4);
  }

  // rows row0 .. row0+63 of [S, D]: into registers
  DEV_INLINE static void load(const short* src, int64_t ss, int row0, int S,
                              int D, s16x8 (&r)[kPer]) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = i * 256 + threadIdx.x;
      const int row = min(row0 + e / kSlots, S - 1);
      const int col = (e % kSlots) * 8;
      r[i] = *reinterpret_cast<const s16x8*>(
          src + static_cast<int64_t>(row) * ss + (col < D ? col : 0));
    }
  }
  // and from registers into LDS, with zeros for what `live` (documents of
  // the 64 rows, negative if there is no such token) and D leave out
  DEV_INLINE static void store(char* lds, const int* live, int D,
                               const s16x8 (&r)[kPer]) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = i * 256 + threadIdx.x;
      const int row = e / kSlots, slot = e % kSlots;
      const s16x8 zero = {0, 0, 0, 0, 0, 0, 0, 0};
      *reinterpret_cast<s16x8*>(lds + at(row, slot)) =
          live[row] >= 0 && slot * 8 < D ? r[i] : zero;
    }
  }

  // left operand: rows row0 + 0..31, columns 16 kk + 0..15
  DEV_INLINE static s16x8 rows(const char* lds, int row0, int kk) {
    const int lane = threadIdx.x % kWave;
    return *reinterpret_cast<const s16x8*>(
        lds + at(row0 + (lane & 31), kk * 2 + (lane >> 5)));
  }
  // transposed left operand: columns 32 db + 0..31 as rows, tokens
  // row0 + 0..15 in the order of the file's head
  DEV_INLINE static s16x8 cols(const char* lds, int row0, int db) {
    const int lane = threadIdx.x % kWave;
    const int i = lane & 15;
    const int row = row0 + ((lane >> 5) << 2) + (i >> 2);
    const int slot = db * 4 + ((lane >> 4) & 1) * 2 + ((i >> 1) & 1);
    const int half = (i & 1) * 8;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s16x4*)(lds + at(row, slot) + half));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s16x4*)(lds + at(row + 8, slot) + half));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

// right operand of an owned token's row: columns 16 kk + 8 h + 0..7
template <int DP>
DEV_INLINE void own_rows(const short* row, bool live, int D,
                         s16x8 (&r)[DP / 16]) {
  const int h = (threadIdx.x % kWave) >> 5;
#pragma unroll
  for (int kk = 0; kk < DP / 16; ++kk) {
    const int col = kk * 16 + h * 8;
    const s16x8 zero = {0, 0, 0, 0, 0, 0, 0, 0};
    r[kk] = live && col < D ? *reinterpret_cast<const s16x8*>(row + col)
                            : zero;
  }
}

// a transposed result: this lane's token gets columns 32 db + (r & 3) +
// 8 (r >> 2) + 4 h
template <typename T, int DP>
DEV_INLINE void store_cols(T* row, const f32x16 (&acc)[DP / 32], float f,
                           bool live, int D) {
  const int h = (threadIdx.x % kWave) >> 5;
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int col = db * 32 + g * 8 + h * 4;
      float x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = live ? acc[db][g * 4 + j] * f : 0.f;
      if (col < D) elem_store4(row + col, x);
    }
}

// summary of one 64-token tile of doc: smallest and largest document, and
// whether there is padding; (INT_MAX, -1) if there is nothing else
__global__ __launch_bounds__(64) void masked_attn_tiles_kernel(
    const int* __restrict__ doc, int4* __restrict__ tiles, int S, int count) {
  const int n = blockIdx.x / count;  // count: tiles a sequence
  const int tok = (blockIdx.x - n * count) * kTile + threadIdx.x;
  const int d = tok < S ? doc[static_cast<int64_t>(n) * S + tok] : 0;
  const bool real = tok < S && d >= 0;
  int lo = real ? d : 0x7fffffff, hi = real ? d : -1;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    lo = min(lo, __shfl_xor(lo, off));
    hi = max(hi, __shfl_xor(hi, off));
  }
  const bool pad = __any(tok < S && d < 0);
  if (threadIdx.x == 0)
    tiles[blockIdx.x] = make_int4(lo, hi, pad, 0);
}

// What the pairs of tokens [q0, q1) x [k0, k1) are: 0 none attended, 1 some,
// 2 all.  A tile that reaches past S counts as mixed on the key side only:
// no query row past S is ever written, or has a statistic but +inf.
DEV_INLINE int meet(bool causal, int prefix, int S, int q0, int q1, int k0,
                    int k1, bool doc, int4 a, int4 b) {
  int c = k1 > S ? 1 : 2;
  const int qe = min(q1, S) - 1, ke = min(k1, S) - 1;
  if (causal) {
    if (k0 > qe && k0 >= prefix) return 0;
    if (!(ke <= q0 || ke < prefix)) c = 1;
  }
  if (doc) {
    if (a.x > b.y || b.x > a.y) return 0;
    if (a.x != a.y || b.x != b.y || a.z || b.z) c = 1;
  }
  return c;
}

DEV_INLINE int4 join(int4 a, int4 b) {
  return make_int4(min(a.x, b.x), max(a.y, b.y), a.z | b.z, 0);
}

// Lists the tiles of [base, base + kList) that meet the owned tokens from own0
// on: (tile << 1) | whole, in order.  Called by the whole workgroup.
template <bool OWN_Q>
DEV_INLINE int list_tiles(const MaskedAttn& a, int n, int own0, int base,
                          int* list, int* count) {
  const int tiles = (a.S + kTile - 1) / kTile;
  __syncthreads();  // the previous list is used up
  if (threadIdx.x < kWave) {
    const int lane = threadIdx.x;
    const int prefix = a.prefix != nullptr ? a.prefix[n] : 0;
    const bool summary = a.tiles != nullptr;
    const int4* row = a.tiles + static_cast<int64_t>(n) * tiles;
    int4 mine = make_int4(0, 0, 0, 0);
    if (summary) {
      const int t = own0 / kTile;
      mine = row[t];
      if (t + 1 < tiles) mine = join(mine, row[t + 1]);
    }
    int found = 0;
    const int end = min(base + kList, tiles);
    for (int t0 = base; t0 < end; t0 += kWave) {
      const int t = t0 + lane;
      int c = 0;
      if (t < end) {
        const int4 other = summary ? row[t] : mine;
        const int s0 = t * kTile;
        c = OWN_Q ? meet(a.causal, prefix, a.S, own0, own0 + kOwn, s0,
                         s0 + kTile, summary, mine, other)
                  : meet(a.causal, prefix, a.S, s0, s0 + kTile, own0,
                         own0 + kOwn, summary, mine, other);
        if (c == 2 && a.doc != nullptr && !summary) c = 1;
      }
      const unsigned long long hit = __ballot(c != 0);
      if (c != 0)
        list[found + __popcll(hit & ((1ull << lane) - 1))] =
            (t << 1) | (c == 2);
      found += __popcll(hit);
    }
    if (lane == 0) *count = found;
  }
  __syncthreads();
  return *count;
}

// document of a token: -1 for padding and past the end, 0 without documents
DEV_INLINE int doc_of(const MaskedAttn& a, int n, int tok) {
  if (tok >= a.S) return -1;
  if (a.doc == nullptr) return 0;
  return max(a.doc[static_cast<int64_t>(n) * a.S + tok], -1);
}

DEV_INLINE const short* row_of(const HeadView& v, int n, int h) {
  return static_cast<const short*>(v.p) + n * v.sn + h * v.sh;
}

// block -> (sequence, head, owned block): one head's blocks stay on one XCD,
// whose L2 then holds what they stream
DEV_INLINE void locate(const MaskedAttn& a, int heads, bool last_first,
                       int* n, int* h, int* own0) {
  const int blocks = (a.S + kOwn - 1) / kOwn;
  const int total = gridDim.x;
  const int q = total / kNumXCD, r = total % kNumXCD;
  const int xcd = blockIdx.x % kNumXCD, idx = blockIdx.x / kNumXCD;
  const int id =
      (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + idx;
  const int nh = id / blocks;
  int b = id % blocks;
  if (last_first) b = blocks - 1 - b;  // causal: the longest rows first
  *n = nh / heads;
  *h = nh % heads;
  *own0 = b * kOwn;
}

// Scores of one 32x32 result, from q.k to base 2, with -inf where masked.
// FIX: the side of the columns.  OWN_Q: columns are queries, rows keys.
// th: tanh of the cap, for the backward.  Returns what is left to multiply
// with (the scale, where nothing before the exponential needs it applied).
struct Score {
  float c;       // scale * log2 e
  float cap_in;  // scale / cap
  float cap_out;  // cap * log2 e
  float slope;   // slope * log2 e
  bool cap, bias, causal;
  int prefix;

  DEV_INLINE Score(const MaskedAttn& a, int n, int h) {
    c = a.scale * kLog2e;
    cap = a.softcap > 0.f;
    cap_in = cap ? a.scale / a.softcap : 0.f;
    cap_out = a.softcap * kLog2e;
    bias = a.slopes != nullptr;
    slope = bias ? a.slopes[h] * kLog2e : 0.f;
    causal = a.causal;
    prefix = a.prefix != nullptr ? a.prefix[n] : 0;
  }

  // own: this lane's token; other0: token of register 0's row for half 0,
  // plus 4 h already added
  template <bool OWN_Q>
  DEV_INLINE void apply(f32x16& z, int own, int own_doc, int other0,
                        const int* other_doc, bool mixed) const {
    if (cap) {
#pragma unroll
      for (int r = 0; r < 16; ++r) z[r] = fast_tanh(z[r] * cap_in) * cap_out;
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r) z[r] *= c;
    }
    if (bias) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        z[r] -= slope * fabsf(static_cast<float>(
                            own - (other0 + (r & 3) + 8 * (r >> 2))));
    }
    if (mixed) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int4 d = *reinterpret_cast<const int4*>(other_doc + g * 8);
        const int dd[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int tok = other0 + g * 8 + j;
          const int qi = OWN_Q ? own : tok, kj = OWN_Q ? tok : own;
          const bool ok = dd[j] == own_doc && dd[j] >= 0 &&
                          (!causal || kj <= qi || kj < prefix);
          if (!ok) z[g * 4 + j] = -INFINITY;
        }
      }
    }
  }
};

template <int DP>
struct Smem {
  char tile[2][2][Tile<DP>::kBytes];  // buffer, operand
  int doc[2][kTile];
  float lse[2][kTile];    // dk/dv only
  float delta[2][kTile];  // dk/dv only
  int list[kList];
  int count;
};

// ---------------------------------------------------------------------------
template <typename T, int DP>
__global__ __launch_bounds__(256, 2) void masked_attn_fwd_kernel(
    MaskedAttn a) {
  using L = Tile<DP>;
  __shared__ __align__(16) Smem<DP> sm;
  int n, h, own0;
  locate(a, a.H, a.causal, &n, &h, &own0);
  const int hk = h / (a.H / a.Hkv);
  const int lane = threadIdx.x % kWave, half = lane >> 5;
  const int own = own0 + (threadIdx.x / kWave) * 32 + (lane & 31);
  const int own_doc = doc_of(a, n, own);
  const bool live = own_doc >= 0;
  const short* kp = row_of(a.k, n, hk);
  const short* vp = row_of(a.v, n, hk);
  s16x8 qf[DP / 16];
  own_rows<DP>(row_of(a.q, n, h) + own * a.q.ss, live, a.D, qf);
  const Score sc(a, n, h);
  f32x16 acc[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) acc[i] = 0.f;
  float m = -INFINITY, l = 0.f;  // l: this half's share

  const int tiles = (a.S + kTile - 1) / kTile;
  for (int base = 0; base < tiles; base += kList) {
    const int count = list_tiles<true>(a, n, own0, base, sm.list, &sm.count);
    s16x8 kr[L::kPer], vr[L::kPer];
    int dr = -1;
    auto fetch = [&](int e) {
      const int t0 = (sm.list[e] >> 1) * kTile;
      L::load(kp, a.k.ss, t0, a.S, a.D, kr);
      L::load(vp, a.v.ss, t0, a.S, a.D, vr);
      if (threadIdx.x < kTile) dr = doc_of(a, n, t0 + threadIdx.x);
    };
    // the documents decide what the tile's rows are stored as: a barrier
    // between them and the rows
    auto keep_doc = [&](int buf) {
      if (threadIdx.x < kTile) sm.doc[buf][threadIdx.x] = dr;
    };
    auto keep = [&](int buf) {
      L::store(sm.tile[buf][0], sm.doc[buf], a.D, kr);
      L::store(sm.tile[buf][1], sm.doc[buf], a.D, vr);
    };
    if (count > 0) {
      fetch(0);
      keep_doc(0);
      __syncthreads();
      keep(0);
      __syncthreads();
    }
    for (int e = 0; e < count; ++e) {
      const int buf = e & 1;
      const bool more = e + 1 < count;
      if (more) fetch(e + 1);
      const int t0 = (sm.list[e] >> 1) * kTile;
      const bool mixed = !(sm.list[e] & 1);
      f32x16 z[2];
      float mx = -INFINITY;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        z[kb] = 0.f;
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)
          z[kb] = mfma<T>(L::rows(sm.tile[buf][0], kb * 32, kk), qf[kk],
                          z[kb]);
        sc.apply<true>(z[kb], own, own_doc, t0 + kb * 32 + 4 * half,
                       sm.doc[buf] + kb * 32 + 4 * half, mixed);
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, z[kb][r]);
      }
      mx = fmaxf(mx, other_half(mx));
      if (__any(mx > m)) {
        const float top = fmaxf(m, mx);
        // a row that has met nothing yet stays at -inf without NaN
        const float f = fast_exp2(m - (top == -INFINITY ? 0.f : top));
        m = top;
        l *= f;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) acc[i] *= f;
      }
      const float top = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          z[kb][r] = fast_exp2(z[kb][r] - top);
          l += z[kb][r];
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          const s16x8 p = round8<T>(z[kb], ks);
#pragma unroll
          for (int db = 0; db < DP / 32; ++db)
            acc[db] = mfma<T>(
                L::cols(sm.tile[buf][1], kb * 32 + ks * 16, db), p, acc[db]);
        }
      }
      if (more) {
        keep_doc(buf ^ 1);
        __syncthreads();
        keep(buf ^ 1);
      }
      __syncthreads();
    }
  }
  l += other_half(l);
  if (own < a.S) {
    T* o = static_cast<T*>(a.o.p) + n * a.o.sn + own * a.o.ss + h * a.o.sh;
    // NaN in a live row's sum is kept: only an empty row is cleared
    const bool clear = !live || l == 0.f;
    store_cols<T, DP>(o, acc, clear ? 0.f : 1.f / l, !clear, a.D);
    if (half == 0)
      a.lse[(static_cast<int64_t>(n) * a.H + h) * a.S + own] =
          clear ? INFINITY : m + log2f(l);
  }
}

// ---------------------------------------------------------------------------
template <typename T, int DP>
__global__ __launch_bounds__(256, 2) void masked_attn_dq_kernel(
    MaskedAttn a) {
  using L = Tile<DP>;
  __shared__ __align__(16) Smem<DP> sm;
  int n, h, own0;
  locate(a, a.H, a.causal, &n, &h, &own0);
  const int hk = h / (a.H / a.Hkv);
  const int lane = threadIdx.x % kWave, half = lane >> 5;
  const int own = own0 + (threadIdx.x / kWave) * 32 + (lane & 31);
  const int own_doc = doc_of(a, n, own);
  const bool live = own_doc >= 0;
  const short* kp = row_of(a.k, n, hk);
  const short* vp = row_of(a.v, n, hk);
  s16x8 qf[DP / 16], gf[DP / 16];
  own_rows<DP>(row_of(a.q, n, h) + own * a.q.ss, live, a.D, qf);
  own_rows<DP>(row_of(a.go, n, h) + own * a.go.ss, live, a.D, gf);
  float delta = 0.f, lse = INFINITY;
  const int64_t stat = (static_cast<int64_t>(n) * a.H + h) * a.S + own;
  {
    s16x8 of[DP / 16];
    own_rows<DP>(row_of(a.o, n, h) + own * a.o.ss, live, a.D, of);
    typedef __attribute__((ext_vector_type(8))) typename Bits16<T>::hw V;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      const V g = __builtin_bit_cast(V, gf[kk]);
      const V o = __builtin_bit_cast(V, of[kk]);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        delta += static_cast<float>(g[j]) * static_cast<float>(o[j]);
    }
    delta += other_half(delta);
    if (own < a.S) {
      lse = a.lse[stat];
      if (half == 0) a.delta[stat] = delta;
    }
  }
  const Score sc(a, n, h);
  f32x16 acc[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) acc[i] = 0.f;

  const int tiles = (a.S + kTile - 1) / kTile;
  for (int base = 0; base < tiles; base += kList) {
    const int count = list_tiles<true>(a, n, own0, base, sm.list, &sm.count);
    s16x8 kr[L::kPer], vr[L::kPer];
    int dr = -1;
    auto fetch = [&](int e) {
      const int t0 = (sm.list[e] >> 1) * kTile;
      L::load(kp, a.k.ss, t0, a.S, a.D, kr);
      L::load(vp, a.v.ss, t0, a.S, a.D, vr);
      if (threadIdx.x < kTile) dr = doc_of(a, n, t0 + threadIdx.x);
    };
    auto keep_doc = [&](int buf) {
      if (threadIdx.x < kTile) sm.doc[buf][threadIdx.x] = dr;
    };
    auto keep = [&](int buf) {
      L::store(sm.tile[buf][0], sm.doc[buf], a.D, kr);
      L::store(sm.tile[buf][1], sm.doc[buf], a.D, vr);
    };
    if (count > 0) {
      fetch(0);
      keep_doc(0);
      __syncthreads();
      keep(0);
      __syncthreads();
    }
    for (int e = 0; e < count; ++e) {
      const int buf = e & 1;
      const bool more = e + 1 < count;
      if (more) fetch(e + 1);
      const int t0 = (sm.list[e] >> 1) * kTile;
      const bool mixed = !(sm.list[e] & 1);
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        f32x16 z = 0.f, dp = 0.f;
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          z = mfma<T>(L::rows(sm.tile[buf][0], kb * 32, kk), qf[kk], z);
          dp = mfma<T>(L::rows(sm.tile[buf][1], kb * 32, kk), gf[kk], dp);
        }
        f32x16 dz;
        if (sc.cap) {
          const f32x16 raw = z;
          sc.apply<true>(z, own, own_doc, t0 + kb * 32 + 4 * half,
                         sm.doc[buf] + kb * 32 + 4 * half, mixed);
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float th = fast_tanh(raw[r] * sc.cap_in);
            dz[r] = fast_exp2(z[r] - lse) * (dp[r] - delta) * (1.f - th * th);
          }
        } else {
          sc.apply<true>(z, own, own_doc, t0 + kb * 32 + 4 * half,
                         sm.doc[buf] + kb * 32 + 4 * half, mixed);
#pragma unroll
          for (int r = 0; r < 16; ++r)
            dz[r] = fast_exp2(z[r] - lse) * (dp[r] - delta);
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          const s16x8 x = round8<T>(dz, ks);
#pragma unroll
          for (int db = 0; db < DP / 32; ++db)
            acc[db] = mfma<T>(
                L::cols(sm.tile[buf][0], kb * 32 + ks * 16, db), x, acc[db]);
        }
      }
      if (more) {
        keep_doc(buf ^ 1);
        __syncthreads();
        keep(buf ^ 1);
      }
      __syncthreads();
    }
  }
  if (own < a.S)
    store_cols<T, DP>(static_cast<T*>(a.gq.p) + n * a.gq.sn + own * a.gq.ss +
                          h * a.gq.sh,
                      acc, a.scale, live, a.D);
}

// ---------------------------------------------------------------------------
template <typename T, int DP>
__global__ __launch_bounds__(256, DP == 128 ? 1 : 2) void
masked_attn_dkv_kernel(MaskedAttn a) {
  using L = Tile<DP>;
  __shared__ __align__(16) Smem<DP> sm;
  int n, hk, own0;
  locate(a, a.Hkv, false, &n, &hk, &own0);
  const int group = a.H / a.Hkv;
  const int lane = threadIdx.x % kWave, half = lane >> 5;
  const int own = own0 + (threadIdx.x / kWave) * 32 + (lane & 31);
  const int own_doc = doc_of(a, n, own);
  const bool live = own_doc >= 0;
  s16x8 kf[DP / 16], vf[DP / 16];
  own_rows<DP>(row_of(a.k, n, hk) + own * a.k.ss, live, a.D, kf);
  own_rows<DP>(row_of(a.v, n, hk) + own * a.v.ss, live, a.D, vf);
  f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) dk[i] = dv[i] = 0.f;

  const int tiles = (a.S + kTile - 1) / kTile;
  for (int base = 0; base < tiles; base += kList) {
    const int count = list_tiles<false>(a, n, own0, base, sm.list, &sm.count);
    // every head of the group over the same list, one after another
    for (int hi = 0; hi < group && count > 0; ++hi) {
      const int h = hk * group + hi;
      const Score sc(a, n, h);
      const short* qp = row_of(a.q, n, h);
      const short* gp = row_of(a.go, n, h);
      const int64_t stat = (static_cast<int64_t>(n) * a.H + h) * a.S;
      s16x8 qr[L::kPer], gr[L::kPer];
      int dr = -1;
      float lr = INFINITY, er = 0.f;
      auto fetch = [&](int e) {
        const int t0 = (sm.list[e] >> 1) * kTile;
        L::load(qp, a.q.ss, t0, a.S, a.D, qr);
        L::load(gp, a.go.ss, t0, a.S, a.D, gr);
        if (threadIdx.x < kTile) {
          const int tok = t0 + threadIdx.x;
          dr = doc_of(a, n, tok);
          lr = tok < a.S ? a.lse[stat + tok] : INFINITY;
          er = tok < a.S ? a.delta[stat + tok] : 0.f;
        }
      };
      auto keep_doc = [&](int buf) {
        if (threadIdx.x < kTile) {
          sm.doc[buf][threadIdx.x] = dr;
          sm.lse[buf][threadIdx.x] = lr;
          sm.delta[buf][threadIdx.x] = er;
        }
      };
      auto keep = [&](int buf) {
        L::store(sm.tile[buf][0], sm.doc[buf], a.D, qr);
        L::store(sm.tile[buf][1], sm.doc[buf], a.D, gr);
      };
      fetch(0);
      keep_doc(0);
      __syncthreads();
      keep(0);
      __syncthreads();
      for (int e = 0; e < count; ++e) {
        const int buf = e & 1;
        const bool more = e + 1 < count;
        if (more) fetch(e + 1);
        const int t0 = (sm.list[e] >> 1) * kTile;
        const bool mixed = !(sm.list[e] & 1);
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) {
          f32x16 z = 0.f, dp = 0.f;
#pragma unroll
          for (int kk = 0; kk < DP / 16; ++kk) {
            z = mfma<T>(L::rows(sm.tile[buf][0], qb * 32, kk), kf[kk], z);
            dp = mfma<T>(L::rows(sm.tile[buf][1], qb * 32, kk), vf[kk], dp);
          }
          const int other = qb * 32 + 4 * half;
          f32x16 th2;
          if (sc.cap) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const float th = fast_tanh(z[r] * sc.cap_in);
              th2[r] = 1.f - th * th;
            }
          }
          sc.apply<false>(z, own, own_doc, t0 + other, sm.doc[buf] + other,
                          mixed);
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const float4 ls = *reinterpret_cast<const float4*>(
                sm.lse[buf] + other + g * 8);
            const float4 de = *reinterpret_cast<const float4*>(
                sm.delta[buf] + other + g * 8);
            const float l4[4] = {ls.x, ls.y, ls.z, ls.w};
            const float d4[4] = {de.x, de.y, de.z, de.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int r = g * 4 + j;
              z[r] = fast_exp2(z[r] - l4[j]);
              dp[r] = z[r] * (dp[r] - d4[j]);
              if (sc.cap) dp[r] *= th2[r];
              z[r] *= kLift<T>;
            }
          }
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) {
            const s16x8 p = round8<T>(z, ks);
            const s16x8 x = round8<T>(dp, ks);
#pragma unroll
            for (int db = 0; db < DP / 32; ++db) {
              dv[db] = mfma<T>(
                  L::cols(sm.tile[buf][1], qb * 32 + ks * 16, db), p, dv[db]);
              dk[db] = mfma<T>(
                  L::cols(sm.tile[buf][0], qb * 32 + ks * 16, db), x, dk[db]);
            }
          }
        }
        if (more) {
          keep_doc(buf ^ 1);
          __syncthreads();
          keep(buf ^ 1);
        }
        __syncthreads();
      }
    }
  }
  if (own < a.S) {
    store_cols<T, DP>(static_cast<T*>(a.gk.p) + n * a.gk.sn + own * a.gk.ss +
                          hk * a.gk.sh,
                      dk, a.scale, live, a.D);
    store_cols<T, DP>(static_cast<T*>(a.gv.p) + n * a.gv.sn + own * a.gv.ss +
                          hk * a.gv.sh,
                      dv, 1.f / kLift<T>, live, a.D);
  }
}

template <typename T, int DP>
void run_fwd(const MaskedAttn& a, hipStream_t stream) {
  const int blocks = (a.S + kOwn - 1) / kOwn;
  masked_attn_fwd_kernel<T, DP>
      <<<a.N * a.H * blocks, 256, 0, stream>>>(a);
}

template <typename T, int DP>
void run_bwd(const MaskedAttn& a, hipStream_t stream) {
  const int blocks = (a.S + kOwn - 1) / kOwn;
  masked_attn_dq_kernel<T, DP><<<a.N * a.H * blocks, 256, 0, stream>>>(a);
  masked_attn_dkv_kernel<T, DP>
      <<<a.N * a.Hkv * blocks, 256, 0, stream>>>(a);
}

template <typename T>
void pick_fwd(const MaskedAttn& a, hipStream_t stream) {
  if (a.D <= 32)
    run_fwd<T, 32>(a, stream);
  else if (a.D <= 64)
    run_fwd<T, 64>(a, stream);
  else
    run_fwd<T, 128>(a, stream);
}

template <typename T>
void pick_bwd(const MaskedAttn& a, hipStream_t stream) {
  if (a.D <= 32)
    run_bwd<T, 32>(a, stream);
  else if (a.D <= 64)
    run_bwd<T, 64>(a, stream);
  else
    run_bwd<T, 128>(a, stream);
}

}  // namespace

void launch_masked_attn_tiles(const MaskedAttn& a, hipStream_t stream) {
  const int tiles = (a.S + kTile - 1) / kTile;
  masked_attn_tiles_kernel<<<tiles * a.N, 64, 0, stream>>>(a.doc, a.tiles,
                                                           a.S, tiles);
}

void launch_masked_attn_fwd(const MaskedAttn& a, Elem type,
                            hipStream_t stream) {
  if (type == Elem::kBF16)
    pick_fwd<bf16>(a, stream);
  else
    pick_fwd<f16>(a, stream);
}

void launch_masked_attn_bwd(const MaskedAttn& a, Elem type,
                            hipStream_t stream) {
  if (type == Elem::kBF16)
    pick_bwd<bf16>(a, stream);
  else
    pick_bwd<f16>(a, stream);
}

}  // namespace colearn
