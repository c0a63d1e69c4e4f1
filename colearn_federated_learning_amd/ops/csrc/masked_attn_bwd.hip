// Masked attention, backward.  The mathematics and the layout stand in
// masked_attn.h.

#include "masked_attn.h"

namespace colearn {

using namespace masked_attn;

namespace {

template <typename T, int DP, Mode M, int KS>
__global__ __launch_bounds__(256, DP == 128 ? 2 : 3) void masked_attn_dq_kernel(
    MaskedAttn a) {
  using L = Tile<DP>;
  constexpr int OWN = 128 / KS, KB = 2 / KS;
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
  const Stream<DP> ks(row_of(a.k, n, hk), a.k.ss);
  const Stream<DP> vs(row_of(a.v, n, hk), a.v.ss);
  s16x8 qf[DP / 16], gf[DP / 16];
  const int there = min(own, a.S - 1);
  own_rows<DP>(row_of(a.q, n, h) + there * a.q.ss, a.D, qf);
  own_rows<DP>(row_of(a.go, n, h) + there * a.go.ss, a.D, gf);
  const int64_t stat = (static_cast<int64_t>(n) * a.H + h) * a.S + own;
  float delta = 0.f, lse = INFINITY;
  const int4* sum;
  {
    s16x8 of[DP / 16], rf[DP / 16];
    own_rows<DP>(row_of(a.o, n, h) + there * a.o.ss, a.D, of);
    own_rows<DP>(static_cast<const short*>(a.rest) +
                     ((static_cast<int64_t>(n) * a.S + there) * a.H + h) * a.D,
                 a.D, rf);
    sum = summary_of(a, n, sm.sum);
    clear<DP>(live, a.D, qf);
    clear<DP>(live, a.D, gf);
    clear<DP>(live, a.D, of);
    clear<DP>(live, a.D, rf);
    typedef __attribute__((ext_vector_type(8))) typename Bits16<T>::hw V;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      const V g = __builtin_bit_cast(V, gf[kk]);
      const V o = __builtin_bit_cast(V, of[kk]);
      const V r = __builtin_bit_cast(V, rf[kk]);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        delta += static_cast<float>(g[j]) *
                 (static_cast<float>(o[j]) + static_cast<float>(r[j]));
    }
    delta += other_half(delta);
    if (own < a.S) lse = a.lse[stat];
  }
  const Score<M> sc(a, h);
  f32x16 acc[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) acc[i] = 0.f;
  Lift<T> lift;

  // probabilities z, 2^up times as large, and dp - delta, of half kb of a tile;
  // w: what the cap takes from dz
  auto scores = [&](int buf, int kb, int t0, bool mixed, float up, f32x16& z,
                    f32x16& dp, f32x16& w) {
    const char* kt = sm.tile[buf][0] + kb * (L::kBytes / 2);
    const char* vt = sm.tile[buf][1] + kb * (L::kBytes / 2);
    const int other = kb * 32 + 4 * half;
    z = 0.f;
    dp = 0.f;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      z = mfma<T>(L::rows(kt, kk), qf[kk], z);
      dp = mfma<T>(L::rows(vt, kk), gf[kk], dp);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) dp[r] -= delta;
    sc.bend(z);
    if constexpr (M == kCap) {
#pragma unroll
      for (int r = 0; r < 16; ++r) w[r] = 1.f - z[r] * z[r];
    }
    const float lane_part =
        sc.c * sc.lean(z, static_cast<float>(own - t0 - other),
                       own_wave - t0 - kb * 32) - lse + up;
    if (mixed) mask<true>(z, own_doc, lim, t0 + other, sm.doc[buf] + other);
#pragma unroll
    for (int r = 0; r < 16; ++r)
      z[r] = fast_exp2(__builtin_fmaf(z[r], sc.c, lane_part));
  };

  settle(qf);
  settle(gf);
  asm volatile("" : "+v"(lse));
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
    if (KS == 2 && tiles <= kList && count == 1) {
      // all that the rows attend to is here: D from p and dp themselves (in
      // the variant of short sequences; in the other it would cost registers)
      float miss = 0.f;
      const int t0 = first_of(entry, base);
      const unsigned cls = (entry >> (4 * (wave / KS))) & 15;
      for (int kb = 0; kb < 2; ++kb) {
        const unsigned c = (cls >> (2 * kb)) & 3;
        if (c == 0) continue;
        f32x16 z, dp, w;
        scores(0, kb, t0, c == 1, 0.f, z, dp, w);
#pragma unroll
        for (int r = 0; r < 16; ++r) miss = __builtin_fmaf(z[r], dp[r], miss);
      }
      delta += miss + other_half(miss);
    }
    for (int e = 0; e < count; ++e) {
      const int buf = e & 1;
      if (e + 1 < count) fetch(buf ^ 1, next);
      const unsigned after = sm.list[min(e + 2, count - 1)];
      const int t0 = first_of(entry, base);
      const unsigned cls = (entry >> (4 * (wave / KS))) & 15;
#pragma unroll
      for (int i = 0; i < KB; ++i) {
        const int kb = KS == 1 ? i : part;
        const unsigned c = (cls >> (2 * kb)) & 3;
        if (c == 0) continue;
        f32x16 z, dp, w;
        scores(buf, kb, t0, c == 1, lift.log2(), z, dp, w);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          dp[r] *= z[r];
          if constexpr (M == kCap) dp[r] *= w[r];
        }
        lift.fit(dp, acc);
        const char* kt = sm.tile[buf][0] + kb * (L::kBytes / 2);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const s16x8 x = round8<T>(dp, s);
#pragma unroll
          for (int db = 0; db < DP / 32; ++db)
            acc[db] = mfma<T>(L::cols(kt, s, db), x, acc[db]);
        }
      }
      if (e + 1 < count) keep(buf ^ 1, next);
      entry = next;
      next = __builtin_amdgcn_readfirstlane(after);
      arrived();
      __syncthreads();
    }
  }
  lift.leave(acc);
  // of the tile buffers: this wave's own part, or its pair's
  char* const mine =
      &sm.tile[0][0][0] +
      (KS == 2 ? (wave / 2) * (DP / 2) * kWave * 4 : wave * DP * kWave);
  if constexpr (KS == 2) {
    float* at = reinterpret_cast<float*>(mine);
    __syncthreads();
    if (part == 1) leave(at, acc);
    __syncthreads();
    if (part == 1) return;
    f32x16 o[DP / 32];
    pick_up(at, o);
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) acc[i] += o[i];
  }
  if (own < a.S && half == 0) a.delta[stat] = delta;
  store_cols<T, DP>(mine,
                    static_cast<T*>(a.gq.p) + n * a.gq.sn + h * a.gq.sh,
                    a.gq.ss, own_wave, a.S, acc, a.scale, live, a.D);
}

// Both sums of 32 keys of size 128 take 128 registers and the keys' own rows
// another 64: one wave a SIMD, with nothing to run while it waits.  KS = 8 is
// for those: two waves a SIMD, eight to a workgroup, in pairs like KS = 2, with
// the own rows in LDS.  Less to run beside a workgroup's begin and end, so for
// long sequences: 8 x 2048 tokens, 16 heads, 678 us, KS = 1 775; 16 x 1024 437
// and 456; 32 x 512, 12 heads, 196 and 184.
constexpr int kEight = 1024;

template <typename T, int DP, Mode M, int KS>
__global__ __launch_bounds__(KS == 8 ? 512 : 256,
                             DP == 128 && KS != 8 ? 1 : 2) void
masked_attn_dkv_kernel(MaskedAttn a) {
  using L = Tile<DP>;
  constexpr bool kLds = KS == 8;
  constexpr int W = kLds ? 8 : 4;
  constexpr int PAIR = kLds ? 2 : KS;  // waves that share 32 owned tokens
  constexpr int OWN = 32 * W / PAIR, KB = 2 / PAIR;
  // Both halves of a tile at once where there is a distance to work out: 1 x
  // 4096 tokens, 12 heads of size 64, 174 us, one after the other 185.
  // Not without (short documents: 78 and 75), nor with the cap (no registers).
  constexpr bool kJoint = KS == 1 && DP <= 64 && M == kBias;
  __shared__ __align__(16) Smem<DP, kLds> sm;
  int n, hs, own0;  // hs: key head and share
  locate<OWN>(a, a.Hkv * a.shares, false, &n, &hs, &own0);
  const int hk = hs / a.shares, share = hs % a.shares;
  // the heads of the group that this workgroup adds up: all, or its share
  const int group = a.H / a.Hkv / a.shares;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave;
  const int half = lane >> 5, part = PAIR == 1 ? 0 : wave & 1;
  const int own_wave = own0 + (wave / PAIR) * 32;
  const int own = own_wave + (lane & 31);
  const int found = doc_of(a, n, own);
  const bool live = found >= 0;
  const int own_doc = live ? found : -2;
  const int lim = pair_limit<false>(a, n, own);
  Docs docs(a, n);
  s16x8 kf[kLds ? 1 : DP / 16], vf[kLds ? 1 : DP / 16];
  const char *kt = nullptr, *vt = nullptr;  // this wave's rows in LDS
  if constexpr (kLds) {
    const Stream<DP, W> ks(row_of(a.k, n, hk), a.k.ss);
    const Stream<DP, W> vs(row_of(a.v, n, hk), a.v.ss);
    for (int i = 0; i < OWN / kTile; ++i) {
      docs.load(own0 + i * kTile, a.S);
      const unsigned long long there = docs.live(own0 + i * kTile, a.S);
      ks.copy(sm.own[0][i], own0 + i * kTile, a.S, a.D, there);
      vs.copy(sm.own[1][i], own0 + i * kTile, a.S, a.D, there);
    }
    kt = sm.own[0][0] + (wave / PAIR) * (L::kBytes / 2);
    vt = sm.own[1][0] + (wave / PAIR) * (L::kBytes / 2);
  } else {
    const int there = min(own, a.S - 1);
    own_rows<DP>(row_of(a.k, n, hk) + there * a.k.ss, a.D, kf);
    own_rows<DP>(row_of(a.v, n, hk) + there * a.v.ss, a.D, vf);
  }
  const int4* sum = summary_of(a, n, sm.sum);
  f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) dk[i] = dv[i] = 0.f;
  Lift<T> lift;

  // N halves of the streamed tile from half qb on; cls: their marks
  auto work = [&](auto number, const Score<M>& sc, int buf, int qb, int t0,
                  unsigned cls) {
    constexpr int N = decltype(number)::value;
    f32x16 zs[N], dps[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const char* qt = sm.tile[buf][0] + (qb + i) * (L::kBytes / 2);
      const char* gt = sm.tile[buf][1] + (qb + i) * (L::kBytes / 2);
      zs[i] = 0.f;
      dps[i] = 0.f;
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        zs[i] = mfma<T>(L::rows(qt, kk), kLds ? L::rows(kt, kk) : kf[kk],
                        zs[i]);
        dps[i] = mfma<T>(L::rows(gt, kk), kLds ? L::rows(vt, kk) : vf[kk],
                         dps[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const char* qt = sm.tile[buf][0] + (qb + i) * (L::kBytes / 2);
      const char* gt = sm.tile[buf][1] + (qb + i) * (L::kBytes / 2);
      const int other = (qb + i) * 32 + 4 * half;
      f32x16& z = zs[i];
      f32x16& dp = dps[i];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 de =
            *reinterpret_cast<const float4*>(sm.delta[buf] + other + g * 8);
        dp[g * 4] -= de.x;
        dp[g * 4 + 1] -= de.y;
        dp[g * 4 + 2] -= de.z;
        dp[g * 4 + 3] -= de.w;
      }
      sc.bend(z);
      if constexpr (M == kCap) {
#pragma unroll
        for (int r = 0; r < 16; ++r) dp[r] *= 1.f - z[r] * z[r];
      }
      const float up = fast_exp2(lift.log2() - kLift<T>);
      sc.lean(z, static_cast<float>(own - t0 - other));
      if (((cls >> (2 * i)) & 3) != 2)
        mask<false>(z, own_doc, lim, t0 + other, sm.doc[buf] + other);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 ls =
            *reinterpret_cast<const float4*>(sm.lse[buf] + other + g * 8);
        const float l4[4] = {ls.x, ls.y, ls.z, ls.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = g * 4 + j;
          z[r] = fast_exp2(__builtin_fmaf(z[r], sc.c, -l4[j]));  // 2^kLift p
          dp[r] *= z[r] * up;
        }
      }
      lift.fit(dp, dk);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const s16x8 p = round8<T>(z, s);
        const s16x8 x = round8<T>(dp, s);
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) {
          dv[db] = mfma<T>(L::cols(gt, s, db), p, dv[db]);
          dk[db] = mfma<T>(L::cols(qt, s, db), x, dk[db]);
        }
      }
    }
  };
  if constexpr (!kLds) {
    clear<DP>(live, a.D, kf);
    clear<DP>(live, a.D, vf);
    settle(kf);
    settle(vf);
  }
  const int tiles = (a.S + kTile - 1) / kTile;
  for (int base = 0; base < tiles; base += kList) {
    const int count = list_tiles<false, OWN / 32>(a, n, own0, base, sum,
                                                  sm.list, &sm.count);
    // every head of the group over the same list, one after another
    for (int hi = 0; hi < group && count > 0; ++hi) {
      const int h = hs * group + hi;
      const Score<M> sc(a, h);
      const Stream<DP, W> qs(row_of(a.q, n, h), a.q.ss);
      const Stream<DP, W> gs(row_of(a.go, n, h), a.go.ss);
      const int64_t stat = (static_cast<int64_t>(n) * a.H + h) * a.S;
      float lr, er;
      auto fetch = [&](int buf, unsigned entry) {
        const int t0 = first_of(entry, base);
        docs.load(t0, a.S);
        if (!(entry & kZeros) && a.D == DP) {
          qs.send(sm.tile[buf][0], t0);
          gs.send(sm.tile[buf][1], t0);
        }
        const int tok =
            min(t0 + static_cast<int>(threadIdx.x) % kTile, a.S - 1);
        lr = a.lse[stat + tok];
        er = a.delta[stat + tok];
      };
      auto keep = [&](int buf, unsigned entry) {
        const int t0 = first_of(entry, base);
        if ((entry & kZeros) || a.D != DP) {
          const unsigned long long live = docs.live(t0, a.S);
          qs.copy(sm.tile[buf][0], t0, a.S, a.D, live);
          gs.copy(sm.tile[buf][1], t0, a.S, a.D, live);
        }
        if (threadIdx.x < kTile) {
          const bool past = t0 + static_cast<int>(threadIdx.x) >= a.S;
          sm.doc[buf][threadIdx.x] = docs.own(t0, a.S);
          sm.lse[buf][threadIdx.x] = past ? INFINITY : lr - kLift<T>;
          sm.delta[buf][threadIdx.x] = past ? 0.f : er;
        }
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
        const unsigned cls = (entry >> (4 * (wave / PAIR))) & 15;
        if constexpr (kJoint) {
          if (cls != 0)
            work(std::integral_constant<int, 2>(), sc, buf, 0, t0, cls);
        } else {
#pragma unroll
          for (int i = 0; i < KB; ++i) {
            const int qb = PAIR == 1 ? i : part;
            const unsigned c = (cls >> (2 * qb)) & 3;
            if (c != 0)
              work(std::integral_constant<int, 1>(), sc, buf, qb, t0, c);
          }
        }
        if (e + 1 < count) keep(buf ^ 1, next);
        entry = next;
        next = __builtin_amdgcn_readfirstlane(after);
        arrived();
        __syncthreads();
      }
    }
  }
  lift.leave(dk);
  // of the tile buffers (KS = 8: and the own rows behind them)
  char* const mine = &sm.tile[0][0][0] +
                     (PAIR == 2 ? (wave / 2) * DP * kWave * 4
                                : wave * DP * kWave);
  if constexpr (PAIR == 2) {
    float* at = reinterpret_cast<float*>(mine);
    __syncthreads();
    if (part == 1) {
      leave(at, dk);
      leave(at + (DP / 2) * kWave, dv);
    }
    __syncthreads();
    if (part == 1) return;
    f32x16 o[DP / 32];
    pick_up(at, o);
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) dk[i] += o[i];
    pick_up(at + (DP / 2) * kWave, o);
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) dv[i] += o[i];
  }
  if (a.shares > 1) {
    if (own >= a.S) return;
    const int64_t size = static_cast<int64_t>(a.N) * a.S * a.Hkv * a.D;
    float* at = a.partial + share * size +
                ((static_cast<int64_t>(n) * a.S + own) * a.Hkv + hk) * a.D;
    put_cols<DP>(at, dk, a.scale, live, a.D);
    put_cols<DP>(at + a.shares * size, dv, fast_exp2(-kLift<T>), live, a.D);
    return;
  }
  store_cols<T, DP>(mine,
                    static_cast<T*>(a.gk.p) + n * a.gk.sn + hk * a.gk.sh,
                    a.gk.ss, own_wave, a.S, dk, a.scale, live, a.D);
  store_cols<T, DP>(mine,
                    static_cast<T*>(a.gv.p) + n * a.gv.sn + hk * a.gv.sh,
                    a.gv.ss, own_wave, a.S, dv, fast_exp2(-kLift<T>), live, a.D);
}

// Shares' sums, four elements a thread: grid.y 0 dk, 1 dv.
template <typename T>
__global__ __launch_bounds__(256) void masked_attn_join_kernel(MaskedAttn a) {
  const int64_t size = static_cast<int64_t>(a.N) * a.S * a.Hkv * a.D;
  const int64_t i =
      (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (i >= size) return;
  const float* p = a.partial + blockIdx.y * a.shares * size + i;
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < a.shares; ++k) {
    float y[4];
    elem_load4(p + k * size, y);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] += y[j];
  }
  const HeadView& v = blockIdx.y == 0 ? a.gk : a.gv;
  const int64_t row = i / a.D;  // (n S + token) Hkv + head
  const int col = static_cast<int>(i - row * a.D);
  const int64_t tok = row / a.Hkv;
  const int h = static_cast<int>(row - tok * a.Hkv);
  const int64_t n = tok / a.S;
  elem_store4(static_cast<T*>(v.p) + n * v.sn + (tok - n * a.S) * v.ss +
                  h * v.sh + col,
              x);
}

struct Backward {
  const MaskedAttn& a;
  hipStream_t stream;

  template <typename T, int DP, Mode M>
  void run() const {
    if (a.S <= kTile || masked_attn_split(a, a.H, 2))
      masked_attn_dq_kernel<T, DP, M, 2>
          <<<a.N * a.H * ((a.S + 63) / 64), 256, 0, stream>>>(a);
    else
      masked_attn_dq_kernel<T, DP, M, 1>
          <<<a.N * a.H * ((a.S + 127) / 128), 256, 0, stream>>>(a);
    const int heads = a.Hkv * a.shares;
    const int blocks = a.N * heads * ((a.S + 127) / 128);
    if (masked_attn_split(a, heads, 1))
      masked_attn_dkv_kernel<T, DP, M, 2>
          <<<a.N * heads * ((a.S + 63) / 64), 256, 0, stream>>>(a);
    else if (DP == 128 && a.S >= kEight)
      masked_attn_dkv_kernel<T, DP, M, DP == 128 ? 8 : 1>
          <<<blocks, 512, 0, stream>>>(a);
    else
      masked_attn_dkv_kernel<T, DP, M, 1><<<blocks, 256, 0, stream>>>(a);
    if (a.shares > 1) {
      const int64_t size = static_cast<int64_t>(a.N) * a.S * a.Hkv * a.D;
      masked_attn_join_kernel<T>
          <<<dim3(static_cast<unsigned>((size / 4 + 255) / 256), 2), 256, 0,
             stream>>>(a);
    }
  }
};

}  // namespace

int masked_attn_shares(const MaskedAttn& a) {
  // Key heads that serve several heads leave the dk/dv grid short: the group
  // is shared out until there are two workgroups a CU, or every head has its
  // own.  2 x 1999 capped tokens, 16 heads over 4, size 128: with the join, 292
  // us in one share, 216 in two, 213 in four.
  const int group = a.H / a.Hkv;
  const int64_t blocks =
      static_cast<int64_t>(a.N) * a.Hkv * ((a.S + 127) / 128);
  for (int k = 1; k < group; ++k)
    if (group % k == 0 && blocks * k >= 2 * kNumCU) return k;
  return group;
}

void launch_masked_attn_bwd(const MaskedAttn& a, Elem type,
                            hipStream_t stream) {
  with_type(Backward{a, stream}, a, type);
}

}  // namespace colearn
