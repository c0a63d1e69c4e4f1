// Masked attention, forward.  The mathematics and the layout stand in
// masked_attn.h.

#include "masked_attn.h"

namespace colearn {

using namespace masked_attn;

namespace {

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
  if (threadIdx.x == 0) tiles[blockIdx.x] = make_int4(lo, hi, pad, 0);
}

template <typename T, int DP, Mode M, int KS>
__global__ __launch_bounds__(256, 2) void masked_attn_fwd_kernel(
    MaskedAttn a) {
  using L = Tile<DP>;
  constexpr int OWN = 128 / KS, KB = 2 / KS;
  __shared__ __align__(16) Smem<DP> sm;
  int n, h, own0;
  locate<OWN>(a, a.H, a.causal, &n, &h, &own0);
  const int hk = h / (a.H / a.Hkv);
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const int half = lane >> 5, part = KS == 1 ? 0 : wave & 1;
  const int own = own0 + (wave / KS) * 32 + (lane & 31);
  const int found = doc_of(a, n, own);
  const bool live = found >= 0;
  const int own_doc = live ? found : -2;
  const int lim = pair_limit<true>(a, n, own);
  const int* doc =
      a.doc != nullptr ? a.doc + static_cast<int64_t>(n) * a.S : nullptr;
  const Stream<DP> ks(row_of(a.k, n, hk), a.k.ss, a.D);
  const Stream<DP> vs(row_of(a.v, n, hk), a.v.ss, a.D);
  s16x8 qf[DP / 16];
  own_rows<DP>(row_of(a.q, n, h) + own * a.q.ss, live, a.D, qf);
  const Score<M> sc(a, h);
  f32x16 acc[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) acc[i] = 0.f;
  float m = -INFINITY, l = 0.f;  // m: of c z; l: this half's share

  const int tiles = (a.S + kTile - 1) / kTile;
  for (int base = 0; base < tiles; base += kList) {
    const int count =
        list_tiles<true, OWN>(a, n, own0, base, sm.list, &sm.count);
    s16x8 kr[L::kPer], vr[L::kPer];
    int dr = -1;
    unsigned rows = 0;
    auto fetch = [&](int e) {
      const int t0 =
          (__builtin_amdgcn_readfirstlane(sm.list[e]) >> 1) * kTile;
      ks.load(t0, a.S, kr);
      vs.load(t0, a.S, vr);
      rows = live_rows<DP>(doc, t0, a.S);
      if (threadIdx.x < kTile) dr = doc_of(a, n, t0 + threadIdx.x);
    };
    auto keep = [&](int buf) {
      Stream<DP>::store(sm.tile[buf][0], rows, a.D, kr);
      Stream<DP>::store(sm.tile[buf][1], rows, a.D, vr);
      if (threadIdx.x < kTile) sm.doc[buf][threadIdx.x] = dr;
    };
    if (count > 0) {
      fetch(0);
      keep(0);
      __syncthreads();
    }
    for (int e = 0; e < count; ++e) {
      const int buf = e & 1;
      const bool more = e + 1 < count;
      const int entry = __builtin_amdgcn_readfirstlane(sm.list[e]);
      if (more) fetch(e + 1);
      const int t0 = (entry >> 1) * kTile;
      f32x16 z[KB];
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < KB; ++i) {
        const int kb = KS == 1 ? i : part;
        const char* kt = sm.tile[buf][0] + kb * (L::kBytes / 2);
        z[i] = 0.f;
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)
          z[i] = mfma<T>(L::rows(kt, kk), qf[kk], z[i]);
      }
#pragma unroll
      for (int i = 0; i < KB; ++i) {
        const int other = (KS == 1 ? i : part) * 32 + 4 * half;
        sc.shape(z[i], static_cast<float>(own - t0 - other));
        if (!(entry & 1))
          mask<true>(z[i], own_doc, lim, t0 + other, sm.doc[buf] + other);
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, z[i][r]);
      }
      mx = fmaxf(mx, other_half(mx)) * sc.c;
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
      for (int i = 0; i < KB; ++i) {
        const int kb = KS == 1 ? i : part;
        const char* vt = sm.tile[buf][1] + kb * (L::kBytes / 2);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          z[i][r] = fast_exp2(__builtin_fmaf(z[i][r], sc.c, -top));
          l += z[i][r];
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const s16x8 p = round8<T>(z[i], s);
#pragma unroll
          for (int db = 0; db < DP / 32; ++db)
            acc[db] = mfma<T>(L::cols(vt, s, db), p, acc[db]);
        }
      }
      if (more) keep(buf ^ 1);
      __syncthreads();
    }
  }
  l += other_half(l);
  if constexpr (KS == 2) {
    constexpr int N = DP / 32;
    float* at = reinterpret_cast<float*>(&sm.tile[0][0][0]) +
                (wave / 2) * (N * 16 + 2) * kWave;
    __syncthreads();  // every list may have been empty
    if (part == 1) {
      leave(at, acc);
      at[N * 16 * kWave + lane] = m;
      at[(N * 16 + 1) * kWave + lane] = l;
    }
    __syncthreads();
    if (part == 1) return;
    f32x16 o[N];
    pick_up(at, o);
    const float m2 = at[N * 16 * kWave + lane];
    const float l2 = at[(N * 16 + 1) * kWave + lane];
    const float top = fmaxf(m, m2);
    const float safe = top == -INFINITY ? 0.f : top;
    const float f = fast_exp2(m - safe), f2 = fast_exp2(m2 - safe);
    m = top;
    l = l * f + l2 * f2;
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = acc[i] * f + o[i] * f2;
  }
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

struct Forward {
  const MaskedAttn& a;
  hipStream_t stream;

  template <typename T, int DP, Mode M>
  void run() const {
    const int heads = a.N * a.H;
    if (masked_attn_split(a, a.H))
      masked_attn_fwd_kernel<T, DP, M, 2>
          <<<heads * ((a.S + 63) / 64), 256, 0, stream>>>(a);
    else
      masked_attn_fwd_kernel<T, DP, M, 1>
          <<<heads * ((a.S + 127) / 128), 256, 0, stream>>>(a);
  }
};

}  // namespace

bool masked_attn_split(const MaskedAttn& a, int heads) {
  const int64_t blocks =
      static_cast<int64_t>(a.N) * heads * ((a.S + 127) / 128);
  return blocks < 2 * kNumCU;
}

void launch_masked_attn_tiles(const MaskedAttn& a, hipStream_t stream) {
  const int tiles = (a.S + kTile - 1) / kTile;
  masked_attn_tiles_kernel<<<tiles * a.N, 64, 0, stream>>>(a.doc, a.tiles,
                                                           a.S, tiles);
}

void launch_masked_attn_fwd(const MaskedAttn& a, Elem type,
                            hipStream_t stream) {
  with_type(Forward{a, stream}, a, type);
}

}  // namespace colearn
