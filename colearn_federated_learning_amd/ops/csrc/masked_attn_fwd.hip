// Masked attention, forward.  The mathematics and the layout stand in
// masked_attn.h.

#include "masked_attn.h"

namespace colearn {

using namespace masked_attn;

namespace {

// summaries of 32 tokens each, two a workgroup; groups: of a sequence
__global__ __launch_bounds__(64) void masked_attn_tiles_kernel(
    const int* __restrict__ doc, int4* __restrict__ tiles, int S,
    int groups) {
  const int pairs = (groups + 1) / 2;
  const int n = blockIdx.x / pairs;
  const int tok = (blockIdx.x - n * pairs) * 64 + threadIdx.x;
  const int4 s = summarise(
      doc[static_cast<int64_t>(n) * S + min(tok, S - 1)], tok < S);
  if (threadIdx.x % 32 == 0 && tok < S)
    tiles[static_cast<int64_t>(n) * groups + tok / 32] = s;
}

template <typename T, int DP, Mode M, int KS>
__global__ __launch_bounds__(256, DP == 128 ? 2 : 3) void masked_attn_fwd_kernel(
    MaskedAttn a) {
  using L = Tile<DP>;
  constexpr int OWN = 128 / KS;
  // Both halves of a tile at once where registers allow it: one's products run
  // under the other's exponentials.  Size 64, 1 x 8192 tokens: 255 us, one
  // after the other 264; size 128: 555 and 552.
  constexpr bool kJoint = KS == 1 && DP <= 64;
  __shared__ __align__(16) Smem<DP> sm;
  int n, h, own0;
  locate<OWN>(a, a.H, a.causal, &n, &h, &own0);
  const int hk = h / (a.H / a.Hkv);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave;
  const int half = lane >> 5, part = KS == 1 ? 0 : wave & 1;
  const int own_wave = own0 + (wave / KS) * 32;
  const int own = own_wave + (lane & 31);
  const int found = doc_of(a, n, own);
  const bool live = found >= 0;
  const int own_doc = live ? found : -2;
  const int lim = pair_limit<true>(a, n, own);
  Docs docs(a, n);
  s16x8 qf[DP / 16];
  own_rows<DP>(row_of(a.q, n, h) + min(own, a.S - 1) * a.q.ss, a.D, qf);
  const int4* sum = summary_of(a, n, sm.sum);
  const Stream<DP> ks(row_of(a.k, n, hk), a.k.ss);
  const Stream<DP> vs(row_of(a.v, n, hk), a.v.ss);
  const Score<M> sc(a, h);
  f32x16 acc[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) acc[i] = 0.f;
  float m = -INFINITY, l = 0.f;  // m: of c z; l: this half's share

  // N x 32 streamed keys from t0 on; cls: their marks, two bits each
  auto work = [&](auto count, const char* kt, const char* vt, const int* dt,
                  int t0, unsigned cls) {
    constexpr int N = decltype(count)::value;
    f32x16 z[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      z[i] = 0.f;
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk)
        z[i] = mfma<T>(L::rows(kt + i * (L::kBytes / 2), kk), qf[kk], z[i]);
    }
    float mx = -INFINITY, lane_part[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int other = t0 + i * 32 + 4 * half;
      sc.bend(z[i]);
      lane_part[i] = sc.c * sc.lean(z[i], static_cast<float>(own - other),
                                    own_wave - t0 - i * 32);
      // a half without any pair comes along as one whose pairs are all masked
      if (((cls >> (2 * i)) & 3) != 2)
        mask<true>(z[i], own_doc, lim, other, dt + i * 32 + 4 * half);
      float hi = z[i][0];
#pragma unroll
      for (int r = 1; r < 16; ++r) hi = fmaxf(hi, z[i][r]);
      mx = fmaxf(mx, __builtin_fmaf(hi, sc.c, lane_part[i]));
    }
    // The sums are kept relative to a maximum that may be outgrown by 2^8
    // before they are scaled anew: p stays within both types' range, and its
    // rounding is relative.
    if (__any(mx > m + 8.f)) {
      const float top = fmaxf(m, fmaxf(mx, other_half(mx)));
      // a row that has met nothing yet stays at -inf without NaN
      const float f = fast_exp2(m - (top == -INFINITY ? 0.f : top));
      m = top;
      l *= f;
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) acc[i] *= f;
    }
    const float top = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        z[i][r] =
            fast_exp2(__builtin_fmaf(z[i][r], sc.c, lane_part[i] - top));
        l += z[i][r];
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const s16x8 p = round8<T>(z[i], s);
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
          acc[db] =
              mfma<T>(L::cols(vt + i * (L::kBytes / 2), s, db), p, acc[db]);
      }
    }
  };
  clear<DP>(live, a.D, qf);
  settle(qf);
  const int tiles = (a.S + kTile - 1) / kTile;
  for (int base = 0; base < tiles; base += kList) {
    const int count = list_tiles<true, OWN / 32>(a, n, own0, base, sum,
                                                 sm.list, &sm.count);
    if (count == 0) continue;
    // what of a tile goes ahead, and what is left for when its turn is near
    auto fetch = [&](int buf, unsigned entry) {
      const int t0 = first_of(entry, base);
      docs.load(t0, a.S);
      if (!(entry & kZeros) && a.D == DP) {
        ks.send(sm.tile[buf][0], t0);
        vs.send(sm.tile[buf][1], t0);
      }
    };
    auto keep = [&](int buf, unsigned entry) {
      const int t0 = first_of(entry, base);
      if ((entry & kZeros) || a.D != DP) {
        const unsigned long long live = docs.live(t0, a.S);
        ks.copy(sm.tile[buf][0], t0, a.S, a.D, live);
        vs.copy(sm.tile[buf][1], t0, a.S, a.D, live);
      }
      if (threadIdx.x < kTile) sm.doc[buf][threadIdx.x] = docs.own(t0, a.S);
    };
    unsigned entry = entry_of(sm.list, 0, count);
    unsigned next = entry_of(sm.list, 1, count);
    fetch(0, entry);
    keep(0, entry);
    arrived();
    __syncthreads();
    for (int e = 0; e < count; ++e) {
      const int buf = e & 1;
      if (e + 1 < count) fetch(buf ^ 1, next);
      const unsigned after = sm.list[min(e + 2, count - 1)];
      const int t0 = first_of(entry, base);
      const char* kt = sm.tile[buf][0];
      const char* vt = sm.tile[buf][1];
      const int* dt = sm.doc[buf];
      const unsigned cls = (entry >> (4 * (wave / KS))) & 15;
      if constexpr (kJoint) {
        if (cls != 0)
          work(std::integral_constant<int, 2>(), kt, vt, dt, t0, cls);
      } else {
#pragma unroll
        for (int i = 0; i < 2 / KS; ++i) {
          const int hf = KS == 2 ? part : i;
          const unsigned c = (cls >> (2 * hf)) & 3;
          if (c != 0)
            work(std::integral_constant<int, 1>(),
                 kt + hf * (L::kBytes / 2), vt + hf * (L::kBytes / 2),
                 dt + hf * 32, t0 + hf * 32, c);
        }
      }
      if (e + 1 < count) keep(buf ^ 1, next);
      entry = next;
      next = __builtin_amdgcn_readfirstlane(after);
      arrived();
      __syncthreads();
    }
  }
  l += other_half(l);
  constexpr int N = DP / 32;
  // of the tile buffers: this wave's own part, or its pair's
  char* const mine = &sm.tile[0][0][0] +
                     (KS == 2 ? (wave / 2) * (N * 16 + 2) * kWave * 4
                              : wave * DP * kWave);
  if constexpr (KS == 2) {
    float* at = reinterpret_cast<float*>(mine);
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
  // NaN in a live row's sum is kept: only an empty row is cleared
  const bool empty = !live || l == 0.f;
  const float f = empty ? 0.f : 1.f / l;
  store_cols<T, DP>(mine,
                    static_cast<T*>(a.o.p) + n * a.o.sn + h * a.o.sh, a.o.ss,
                    own_wave, a.S, acc, f, !empty, a.D);
  if (a.rest != nullptr) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float x = acc[i][r] * f;
        acc[i][r] = x - elem_round(x, static_cast<const T*>(nullptr));
      }
    const int64_t row = static_cast<int64_t>(a.H) * a.D;
    store_cols<T, DP>(mine,
                      static_cast<T*>(a.rest) + n * a.S * row + h * a.D, row,
                      own_wave, a.S, acc, 1.f, !empty, a.D);
  }
  if (own < a.S && half == 0)
    a.lse[(static_cast<int64_t>(n) * a.H + h) * a.S + own] =
        empty ? INFINITY : m + log2f(l);
}

struct Forward {
  const MaskedAttn& a;
  hipStream_t stream;

  template <typename T, int DP, Mode M>
  void run() const {
    const int heads = a.N * a.H;
    if (a.S <= kTile || masked_attn_split(a, a.H, 2))
      masked_attn_fwd_kernel<T, DP, M, 2>
          <<<heads * ((a.S + 63) / 64), 256, 0, stream>>>(a);
    else
      masked_attn_fwd_kernel<T, DP, M, 1>
          <<<heads * ((a.S + 127) / 128), 256, 0, stream>>>(a);
  }
};

}  // namespace

bool masked_attn_split(const MaskedAttn& a, int heads, int per_cu) {
  const int64_t blocks =
      static_cast<int64_t>(a.N) * heads * ((a.S + 127) / 128);
  return blocks < per_cu * kNumCU;
}

void launch_masked_attn_tiles(const MaskedAttn& a, hipStream_t stream) {
  const int groups = (a.S + 31) / 32;
  masked_attn_tiles_kernel<<<(groups + 1) / 2 * a.N, 64, 0, stream>>>(
      a.doc, a.tiles, a.S, groups);
}

void launch_masked_attn_fwd(const MaskedAttn& a, Elem type,
                            hipStream_t stream) {
  with_type(Forward{a, stream}, a, type);
}

}  // namespace colearn
