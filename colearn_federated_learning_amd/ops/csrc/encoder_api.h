// Launchers of the encoder-training kernels (adamw.hip, add_norm.hip,
// masked_attn_fwd.hip, masked_attn_bwd.hip), shared with bindings_encoder.cpp.
#pragma once

#include <hip/hip_runtime_api.h>

#include <cstdint>

namespace colearn {

enum class Elem : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

// ---- AdamW over many tensors ----------------------------------------------
constexpr int kAdamwTensors = 48;   // tensors a launch; the table is passed by
                                    // value and has to fit 4 KB of arguments
constexpr int kAdamwBlock = 256;    // elements that share one 8-bit scale
constexpr int kAdamwChunk = 1024;   // elements a workgroup: a block a wave

struct AdamwTensor {
  void* p;
  const void* g;
  void* m;  // fp32, or e4m3 codes
  void* v;  // fp32, or e4m3 codes of the root
  float* ms;
  float* vs;  // scales, one a block (8-bit only)
  const float* ref;
  int64_t n;
};

struct AdamwTable {
  AdamwTensor t[kAdamwTensors];
  float keep[kAdamwTensors];       // 1 - lr * weight decay
  int first[kAdamwTensors + 1];    // first workgroup of each tensor
  unsigned long long aligned;      // bit i: tensor i takes vector accesses
  int count;
};

struct AdamwScalars {
  float b1, omb1, b2, omb2, eps, mu, step, inv_bc2;
  const float* live;  // [step, inv_bc2] on the device, or null
};

void launch_adamw(const AdamwTable& t, const AdamwScalars& s, bool p_bf16,
                  bool g_bf16, bool eight, bool prox, hipStream_t stream);

// ---- residual add + layer norm ----------------------------------------------
constexpr int kAddNormMaxH = 16384;

struct AddNormFwd {
  const void* x;
  const void* r;  // or null
  const float* w;
  const float* b;
  void* s;  // written if r is there
  void* y;
  float* mean;
  float* inv;
  int64_t rows;
  int groups, H;
  float eps;
};

struct AddNormBwd {
  const void* gy;
  const void* gs;  // gradient of the sum itself, or null
  const void* s;
  const float* w;
  const float* mean;
  const float* inv;
  void* gx;
  float* dw;
  float* db;
  float* partials;  // [groups][parts][2][H]
  int64_t rows;
  int groups, H, parts;
};

int add_norm_parts(int64_t rows, int groups, int H);
void launch_add_norm_fwd(const AddNormFwd& f, Elem type, bool vec,
                         hipStream_t stream);
void launch_add_norm_bwd(const AddNormBwd& b, Elem type, bool vec,
                         hipStream_t stream);

// ---- masked attention ---------------------------------------------------------
constexpr int kAttnTile = 64;     // streamed tokens a tile
constexpr int kAttnGroup = 32;    // tokens an entry of the mask's summary
constexpr int kAttnShort = 1024;  // up to here workgroups make their own

struct HeadView {  // [N, S, heads, D] with D contiguous
  void* p;
  int64_t sn, ss, sh;
};

struct MaskedAttn {
  HeadView q, k, v, o;        // o: [N, S, H, D]
  HeadView go, gq, gk, gv;    // backward only
  // What rounding took from o, in o's type and [N, S, H, D]; null if no
  // backward pass follows.
  void* rest;
  const int* doc;             // [N, S], or null
  const int* prefix;          // [N], or null
  const float* slopes;        // [H], or null
  int4* tiles;                // [N, ceil(S / 32)] summary of doc, or null
  float* lse;                 // [N, H, S], base 2; +inf for empty rows
  float* delta;               // [N, H, S], backward only
  float* partial;             // [2, shares, N, S, Hkv, D], if shares > 1
  int shares;                 // of a key head's heads, backward only
  int N, S, H, Hkv, D;
  bool causal;
  float scale, softcap;
};

// Whether two waves share 32 owned tokens: if `heads` a sequence and 128 tokens
// a workgroup make fewer than per_cu workgroups a CU.  Both sides measured,
// 12 heads of size 64, us with two waves / with one: forward 1 x 4096 tokens
// (384 workgroups) 79 / 94, 2 x 4096 (768) 161 / 136; dq 98 / 117 and
// 198 / 172; dk/dv 1 x 2048 (192) 46 / 56, 1 x 4096 (384) 155 / 141.
// The forward and dq also do for sequences of up to 64 tokens, where half of a
// workgroup's 128 would be past the end: 2048 x 32 forward 228 / 250.  dk/dv
// does not: 369 / 337.
bool masked_attn_split(const MaskedAttn& a, int heads, int per_cu);
// into how many shares dk/dv divides the heads of a key head
int masked_attn_shares(const MaskedAttn& a);
void launch_masked_attn_tiles(const MaskedAttn& a, hipStream_t stream);
void launch_masked_attn_fwd(const MaskedAttn& a, Elem type,
                            hipStream_t stream);
void launch_masked_attn_bwd(const MaskedAttn& a, Elem type,
                            hipStream_t stream);

}  // namespace colearn
