// Causal GQA attention of a step's query rows over the dense 8-bit block KV
// cache (layout: fdms_block_kv.h), single tokens and longer query runs.
//
// Sequence b has query rows cu[b] .. cu[b+1] - 1, the last of its context[b]
// keys: query i of n sees keys 0 .. context - n + i.  With codes k, v of scales
// sK, sV (per block and head)
//
//   s_ij = scale * sK_j * <q_i, k_j>     p_ij = exp(s_ij - max_j s_ij)
//   o_i  = sum_j p_ij sV_j v_j / sum_j p_ij
//
// both products on v_mfma_f32_16x16x32_f16 with the codes as halves (exact).
// Taking S^T = K Q^T and O^T = V^T P^T, a lane (g = lane / 16, c = lane % 16)
// owns one query, column c, in both: its maximum, sum and rescale factors are
// scalars of the lane.  The 16 key rows of a score product are free to choose;
// product t of four takes tokens 4t .. 4t + 3 of each of four tiles, so lane
// group g ends up with the 16 tokens of tile g in registers, and that is what
// the second product wants of it: no shuffle and no LDS between the two, and K
// and V go from memory straight to the operand registers.
//
// P goes to halves, not bf16: 2^-11 of each weight, so that the result's own
// rounding to bf16 (2^-8) stays the error there is.  Row sums stay in fp32, of the
// unrounded weights in the kernel for few rows and of the rounded ones (which the
// numerator has) in the one for many.
#include <cmath>
#include <type_traits>

#include "fdms_block_kv.h"

namespace fdms {

constexpr int kGroupKeys = 64;  // keys a wave takes at once: four tiles
constexpr int kMaxSplits = 256;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kNegInf = -__builtin_huge_valf();

struct BlockAttnArgs {
  const void* q;
  int64_t qs_t, qs_h;
  void* out;
  int64_t os_t, os_h;
  const uint8_t* kc;
  int64_t kc_b, kc_h;
  const uint8_t* vc;
  int64_t vc_b, vc_h;
  const float* k_scale;
  const float* v_scale;
  int64_t sc_b;
  const int32_t* tables;
  int64_t bt_b;
  const int32_t* context;
  const int32_t* cu;  // nullptr: one query row per sequence
  // Parts of a row that several splits share: [split][...][head][D] unnormalised
  // and [split][...][head][2], its maximum and sum.  Of the kernel for few rows
  // by (sequence, query), of the one for many by row of q.
  float *few_o, *few_ml, *part_o, *part_ml;
  int* part_used;   // [row of q][head]: splits of the second kernel that hold a part of it (0 or 1: none)
  int width, num_blocks, shift, num_seqs, num_kv_heads, group, total_rows;
  int few_rows;     // sequences of at most so many rows are block_attn_kernel's, longer ones the tile kernel's
  int q_f16;
  float scale;
};

// Sequence b's query rows and keys, cut to what q and the table row can hold.
struct SeqSpan {
  int q0, n, ctx;
};
__device__ __forceinline__ SeqSpan seq_span(const BlockAttnArgs& a, int b) {
  SeqSpan s;
  s.q0 = a.cu ? max(a.cu[b], 0) : b;
  s.n = (a.cu ? min(a.cu[b + 1], a.total_rows) : b + 1) - s.q0;
  s.ctx = (int)min((int64_t)max(a.context[b], 0), (int64_t)a.width << a.shift);
  return s;
}

// The splits a query tile uses of the launch's: of about `share` 64-key groups
// each, so a short context leaves the rest of its workgroups idle and a batch of
// unequal ones is cut into equal pieces.
__device__ __forceinline__ int splits_used(int groups, int splits, int share) {
  return min(splits, max(1, (groups + share - 1) / share));
}

// Where a split's part of (row t of q, head) lies, in rows of D (part_o) or 2
// (part_ml), and that of query i of sequence b in few_o and few_ml.
__device__ __forceinline__ int64_t part_row(const BlockAttnArgs& a, int split, int t, int head) {
  return ((int64_t)split * a.total_rows + t) * (a.num_kv_heads * a.group) + head;
}
__device__ __forceinline__ int64_t few_row(const BlockAttnArgs& a, int split, int b, int i, int head) {
  return (((int64_t)split * a.num_seqs + b) * a.few_rows + i) * (a.num_kv_heads * a.group) + head;
}

__device__ __forceinline__ void store_out4(void* out, int64_t at, f32x4_t v, int f16) {
  typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
  const u32x2_t h = __builtin_bit_cast(u32x2_t, __builtin_convertvector(v, f16x4_t));
  const u32x2_t b = __builtin_bit_cast(u32x2_t, __builtin_convertvector(v, bf16x4_t));  // v_cvt_pk_bf16_f32
  const u32x2_t r = f16 ? h : b;
  *(u32x2_t*)((uint16_t*)out + at) = r;
}

// Eight fp16 or bf16 values; both read without a branch.
__device__ __forceinline__ void halves_to_f32(u32x4_t raw, int f16, float* x) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t e = raw[j >> 1] >> (16 * (j & 1));
    const float as_half = (float)__builtin_bit_cast(f16_t, (uint16_t)e), as_bf16 = bf16_to_f32(e & 0xFFFFu);
    x[j] = __uint_as_float(f16 ? __float_as_uint(as_half) : __float_as_uint(as_bf16));
  }
}

// Power of two that brings a row of largest magnitude amax near 2^14, so the
// row's bf16 values are halves exactly down to 2^-31 of the largest.  Rows of
// zeros, infinities or NaN are left as they are.
__device__ __forceinline__ float q_factor(float amax) {
  const int e = (int)(__float_as_uint(amax) >> 23) - 127;
  if (!(amax > 0.0f) || e > 127) return 1.0f;
  return __uint_as_float((uint32_t)(min(14 - e, 126) + 127) << 23);
}

// Sequences of few query rows (row r: token r / group, head r % group of the kv
// head; at most 16 * MT).  One workgroup takes all of them over one split of
// the keys; its four waves take 64-key groups in turn and join at the end.
//
// Bound by HBM for a loaded server (64 sequences of 293 000 tokens, 8 kv heads of
// 128, int8: 143 us and 5 for the join, 4.1 TB/s), by the chain of loads (lengths,
// block ids, codes) for a few sequences (one of 8 000 tokens, head_dim 64: 5.6 + 3.6
// us).  Cutting contexts into equal pieces, instead of a fixed count each, took
// the first from 207 to 164 us, the next keys' loads under way while these are
// multiplied to 146; pieces of at most 1 024, 2 048 and 4 096 keys 152, 147 and
// 149.  On the kernel for many rows the same batch takes 284 us at best, eight
// sequences of 50 000 tokens 50 against 29, and 20 rows (five drafted tokens of 4
// heads) 85 against 56.
// (three or four waves per SIMD with 16 rows, two with 32)
template <int D, int MT>
constexpr int kFewWaves = MT == 1 ? (D == 64 ? 4 : 3) : 2;

template <int D, bool FP8, int MT>
__global__ __launch_bounds__(256, (kFewWaves<D, MT>)) void block_attn_kernel(const BlockAttnArgs a, int splits, int share) {
  constexpr int KL = D / 64, DC = D / 16, KS = D / 32;  // K loads per row and lane, V row groups, K steps
  constexpr int ROWS = 16 * MT, PAD = D + 4;
  __shared__ float s_o[4][ROWS][PAD];
  __shared__ float s_ml[4][ROWS][2];
  const int pairs = a.num_seqs * a.num_kv_heads;
  const int pair = blockIdx.x % pairs, split = blockIdx.x / pairs;
  const int b = pair / a.num_kv_heads, h = pair % a.num_kv_heads;
  const SeqSpan sp = seq_span(a, b);
  if (sp.n <= 0 || sp.n > a.few_rows) return;
  const int rows = sp.n * a.group;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, c = lane & 15;
  const int first_vis = sp.ctx - sp.n + 1;  // keys query 0 sees
  const int keys = sp.ctx, full = first_vis;  // keys that the last query sees, and that all of them see
  const int groups = (keys + kGroupKeys - 1) / kGroupKeys;
  const int used = splits_used(groups, splits, share);
  if (split >= used) return;
  const int per = (groups + used - 1) / used;
  const int g_end = min(groups, (split + 1) * per);

  // Q^T operand: lane (g, c) holds channels a * 64 + g * 16 + 8 * half .. + 7 of row c
  f16x8_t qf[MT][KS];
  float qmul[MT];  // score factor of the lane's row
  int vis[MT];     // keys it sees
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int r = m * 16 + c;
    const bool on = r < rows;
    const int i = on ? r / a.group : 0, hq = h * a.group + (on ? r % a.group : 0);
    vis[m] = on ? min(sp.ctx, first_vis + i) : 0;
    const int64_t at = (int64_t)(sp.q0 + i) * a.qs_t + (int64_t)hq * a.qs_h;
    float x[KS][8], amax = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const u32x4_t raw = *(const u32x4_t*)((const uint16_t*)a.q + at + (s >> 1) * 64 + g * 16 + (s & 1) * 8);
      halves_to_f32(raw, a.q_f16, x[s]);
#pragma unroll
      for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(x[s][j]));
    }
    const float f = q_factor(rows_max(amax));
    qmul[m] = (a.scale * kLog2e) * (1.0f / f);
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) qf[m][s][j] = (f16_t)(x[s][j] * f);
  }

  f32x4_t o[MT][DC];
  float mx[MT], l[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    mx[m] = kNegInf;
    l[m] = 0.0f;
#pragma unroll
    for (int d = 0; d < DC; ++d) o[m][d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }
  float sref = 1.17549435e-38f;  // the largest V scale so far: P * sV / sref stays in a half's range

  const int32_t* row_table = a.tables + (int64_t)b * a.bt_b;
  const uint8_t* kbase = a.kc + (int64_t)h * a.kc_h;
  const uint8_t* vbase = a.vc + (int64_t)h * a.vc_h;
  const int bmask = (1 << a.shift) - 1;

  // The lane's V tile is g, that of its K rows c / 4.  Ids are loaded a step
  // ahead of codes and scales, and a step's K as soon as the score product has
  // taken the last one's, its V after the second product: the registers that hold
  // one step's codes have the next one's on their way.
  auto id_at = [&](int gi, int quarter) {  // as loaded; a step past the end reads its last one's
    const int key = min(gi, g_end - 1) * kGroupKeys + 16 * quarter;
    return row_table[min(key, keys - 1) >> a.shift];
  };
  auto there = [&](int gi, int quarter, int id) { return gi * kGroupKeys + 16 * quarter < keys && id >= 0 && id < a.num_blocks; };
  u32x4_t kr[4][KL], vr[DC];
  auto load_k = [&](int gi, int id) {
    const int row = ((gi * kGroupKeys + 16 * (c >> 2)) & bmask) + (c & 3);
    const uint8_t* p = kbase + (int64_t)id * a.kc_b + row * D + g * 16;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int x = 0; x < KL; ++x) kr[t][x] = *(const u32x4_t*)(p + 4 * t * D + 64 * x);
  };
  auto load_v = [&](int gi, int id) {
    const uint8_t* p = vbase + (int64_t)id * a.vc_b + ((gi * kGroupKeys + 16 * g) & bmask) * D + c * kTile;
#pragma unroll
    for (int d = 0; d < DC; ++d) vr[d] = *(const u32x4_t*)(p + 256 * d);
  };
  const int gi0 = split * per + wave;
  float sk_n = 0.0f, sv_n = 0.0f;
  int idk_n = 0, idv_n = 0;
  bool okv_n = false;
  if (gi0 < g_end) {
    const int ik = id_at(gi0, c >> 2), iv = id_at(gi0, g);
    idk_n = id_at(gi0 + 4, c >> 2);
    idv_n = id_at(gi0 + 4, g);
    okv_n = there(gi0, g, iv);
    const int id = okv_n ? iv : 0;
    load_k(gi0, there(gi0, c >> 2, ik) ? ik : 0);
    sk_n = a.k_scale[(int64_t)id * a.sc_b + h];
    sv_n = a.v_scale[(int64_t)id * a.sc_b + h];
    load_v(gi0, id);
  }
  for (int gi = gi0; gi < g_end; gi += 4) {
    const int key0 = gi * kGroupKeys, kv_v = key0 + 16 * g;
    const bool okv = okv_n;
    const float sk = okv ? sk_n : 0.0f, sv = okv ? sv_n : 0.0f;
    // the next step's blocks (the last step's own once more where there is none)
    const int gn = min(gi + 4, g_end - 1);
    okv_n = there(gn, g, idv_n);
    const int idk = there(gn, c >> 2, idk_n) ? idk_n : 0, idv = okv_n ? idv_n : 0;
    f32x4_t st[MT][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int m = 0; m < MT; ++m) st[m][t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const f16x8_t kf = codes8_to_f16<FP8>(kr[t][s >> 1][2 * (s & 1)], kr[t][s >> 1][2 * (s & 1) + 1]);
#pragma unroll
        for (int m = 0; m < MT; ++m)
          st[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[m][s], st[m][t], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);  // or all codes are converted, into registers of their own, first
    }
    load_k(gn, idk);
    sk_n = a.k_scale[(int64_t)idv * a.sc_b + h];
    sv_n = a.v_scale[(int64_t)idv * a.sc_b + h];
    idk_n = id_at(gi + 8, c >> 2);
    idv_n = id_at(gi + 8, g);
    __builtin_amdgcn_sched_barrier(0);
    const int live = okv ? keys - kv_v : 0;  // of the lane's tile; rows past it hold whatever the block held
    const float sv_top = rows_max(sv);
    float osc = 1.0f;
    if (sv_top > sref) {
      osc = sref / sv_top;
      sref = sv_top;
    }
    const float vmul = sv / sref;
    const bool masked = __any(!okv) || key0 + kGroupKeys > full;

    f16x8_t pf[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const float mul = qmul[m] * sk;
      float top = kNegInf;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma clang fp contract(off)
          float x = st[m][t][r] * mul;  // rounded, as the maximum taken of it is
          if (masked && !(okv && kv_v + 4 * t + r < vis[m])) x = kNegInf;
          st[m][t][r] = x;
          top = fmaxf(top, x);
        }
      const float mnew = fmaxf(mx[m], rows_max(top));
      const float base = mnew == kNegInf ? 0.0f : mnew;
      const float alpha = __builtin_amdgcn_exp2f(mx[m] - base);
      mx[m] = mnew;
      float sum = 0.0f;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        f32x4_t p;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          p[r] = __builtin_amdgcn_exp2f(st[m][t][r] - base);
          sum += p[r];
          p[r] *= vmul;
        }
        const f16x4_t ph = __builtin_convertvector(p, f16x4_t);
#pragma unroll
        for (int r = 0; r < 4; ++r) pf[m][t >> 1][4 * (t & 1) + r] = ph[r];
      }
      l[m] = l[m] * alpha + sum;
      const float f = alpha * osc;
#pragma unroll
      for (int d = 0; d < DC; ++d) o[m][d] *= f;
    }
    if constexpr (FP8) {
      // a byte of an unwritten row may be a NaN code, and 0 * NaN is no 0
      if (__any(live < kTile)) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int nb = min(max(live - 4 * w, 0), 4);
          const uint32_t keep = nb == 4 ? 0xFFFFFFFFu : (1u << (8 * nb)) - 1u;
#pragma unroll
          for (int d = 0; d < DC; ++d) vr[d][w] &= keep;
        }
      }
    }
#pragma unroll
    for (int d = 0; d < DC; ++d) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const f16x8_t vf = codes8_to_f16<FP8>(vr[d][2 * u], vr[d][2 * u + 1]);
#pragma unroll
        for (int m = 0; m < MT; ++m) o[m][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[m][u], o[m][d], 0, 0, 0);
      }
      if (d & 1) __builtin_amdgcn_sched_barrier(0);
    }
    load_v(gn, idv);
  }

  // join the four waves: every partial to the workgroup's maximum
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const float sum = rows_sum(l[m]);
    if (g == 0) {
      s_ml[wave][m * 16 + c][0] = mx[m];
      s_ml[wave][m * 16 + c][1] = sum;
    }
#pragma unroll
    for (int d = 0; d < DC; ++d) *(f32x4_t*)&s_o[wave][m * 16 + c][16 * d + 4 * g] = o[m][d] * sref;
  }
  __syncthreads();
  for (int e = tid; e < ROWS * (D / 4); e += 256) {
    const int r = e / (D / 4), d = (e % (D / 4)) * 4;
    if (r >= rows) break;
    const int t = sp.q0 + r / a.group, head = h * a.group + r % a.group;
    float top = kNegInf;
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, s_ml[w][r][0]);
    const float base = top == kNegInf ? 0.0f : top;
    float sum = 0.0f;
    f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(s_ml[w][r][0] - base);
      sum += s_ml[w][r][1] * f;
      v += *(const f32x4_t*)&s_o[w][r][d] * f;
    }
    if (used == 1) {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // a row that sees no key: zeros
      store_out4(a.out, (int64_t)t * a.os_t + (int64_t)head * a.os_h + d, v * inv, a.q_f16);
    } else {
      const int64_t at = few_row(a, split, b, r / a.group, head);
      *(f32x4_t*)(a.few_o + at * D + d) = v;
      if (d == 0) {
        a.few_ml[2 * at] = top;
        a.few_ml[2 * at + 1] = sum;
      }
    }
    if (a.part_used && split == 0 && d == 0) a.part_used[part_row(a, 0, t, head)] = 0;
  }
}

// Sequences of many query rows: 32 rows of a kv head (32 / group tokens, all of
// the group's heads) per wave over one split of the keys, NW waves a workgroup.
//
// 64 keys at a time go from the cache to LDS as halves, converted once by the
// workgroup's waves and read by each of them; two buffers each of K and V, one
// barrier per 64 keys.  v_mfma_f32_32x32x16_f16 with S^T = K Q^T, O^T = V^T P^T:
// a lane owns one query (column lane % 32).  V's 16 tokens are written in the
// order in which a lane of a score tile holds them (0-3, 8-11, 4-7, 12-15), so
// P goes from one product to the other in registers.
//
// Measured: 777 queries over 30 788 tokens, 32 / 8 heads of 128, int8, 457 us with
// the join (847 TFLOP/s); four prompts of 17 127 tokens, head_dim 64, e4m3fn, 480
// us (677).  Of the first case's cycles, at the 1.8 GHz that the clock falls to,
// the matrix cores are busy 43 %, the vector unit 62 % and LDS 43 %: products and
// vector work share a wave's issue, and no part dominates (with the scale factors,
// the conversions, the exponentials or the maxima left out it takes 442, 386, 425,
// 438 us).  Steps on the way, first / second case: products, conversion, softmax,
// products one after another 510 / 850; pipelined as below 495 / 705; in a set order
// 450 / 711; sequences turned with the tile 455 / 490.  Eight waves on 256 rows,
// which halves the conversions, 459 / 569: the workgroup's one barrier then holds
// up the whole CU.
//
// The matrix cores and the vector unit are about equally loaded (the
// exponentials, and the conversion of the codes), so they have to run at the
// same time: step t's exponentials stand beside the product of step t + 1's
// keys, the conversion of step t + 2's K and t + 1's V beside step t's P V.  The
// codes come from memory one step before they are converted, block ids one step
// before those.
//
// The blocks' scales go into the halves: a block's codes times its scale over
// the largest so far (a power of two no greater than 1 for the store's scales;
// other ratios are rounded to a half, and the products with them).
// What falls below a half's range there is 2^-25 of that largest scale, far less
// than the fp32 sum it joins can hold next to it.  Then one factor holds for all
// keys of a step, and exp(s - max) is one fma and one v_exp_f32 per score.
//
// A row's maximum is raised only when a score passes it by 2^8 (P stays below
// 2^8, in a half's range): O is rescaled in the first steps and hardly again.
constexpr int kTileWaves = 4, kTileRows = 32 * kTileWaves;
constexpr float kLazyMax = 8.0f;

__device__ __forceinline__ float half_max(float v) {  // over lanes l, l ^ 32
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Four codes as halves times a factor.
template <bool FP8>
__device__ __forceinline__ u32x2_t codes_scaled(uint32_t c, f16x2_t f) {
  u32x2_t r;
  uint32_t lo, hi;
  codes_to_f16<FP8>(c, &lo, &hi);
  r[0] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, lo) * f);
  r[1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, hi) * f);
  return r;
}

__device__ __forceinline__ float quad_max(float v) {  // over the four tiles, the same for the wave (a scalar register)
  v = fmaxf(v, dpp_mov_f<0xB1>(v));
  v = fmaxf(v, dpp_mov_f<0x4E>(v));
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
}

// The larger of two scalars that are not negative (or NaN), whose bits order as they do: stays in scalar registers.
__device__ __forceinline__ float scalar_max(float a, float b) {
  return __builtin_bit_cast(float, max(__builtin_bit_cast(int, a), __builtin_bit_cast(int, b)));
}

// 16-byte chunk c of row r of a K step (2 D bytes a row) or V step (128 bytes)
// lies at slot c ^ swizzle(r): 16 rows' chunks c spread over the 64 LDS banks.
template <int BYTES>
__device__ __forceinline__ int lds_swizzle(int row) {
  return BYTES == 256 ? row & 15 : (row >> 1) & 7;
}

template <int D, bool FP8>
__global__ __launch_bounds__(64 * kTileWaves, 2) void block_attn_tile_kernel(const BlockAttnArgs a, int splits) {
  constexpr int KSTEP = D / 16, DT = D / 32, KP = D / 64, ROWS = kTileRows;
  constexpr int KB = 64 * D * 2;          // bytes of a step's K or V in LDS
  __shared__ __align__(16) uint8_t s_kv[4 * KB];  // K, K, V, V
  const int pairs = a.num_seqs * a.num_kv_heads;
  const int pair = blockIdx.x % pairs, split = blockIdx.x / pairs;
  // Consecutive workgroups go to the XCDs in turn, and on an XCD to its shader
  // engines in turn: the head stays the fastest index (a head's tiles share
  // its K and V in one L2), and the sequence turns with the tile, or one engine
  // would get all tiles of the longest sequence.
  const int b = (int)((pair / a.num_kv_heads + blockIdx.y) % (unsigned)a.num_seqs), h = pair % a.num_kv_heads;
  const SeqSpan sp = seq_span(a, b);
  if (sp.n <= a.few_rows) return;
  const int rows = sp.n * a.group, tiles = (rows + ROWS - 1) / ROWS;
  const int tile = tiles - 1 - (int)blockIdx.y;  // the tiles that see most keys first
  if (tile < 0) return;
  const int row0 = tile * ROWS;
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, c = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int first_vis = sp.ctx - sp.n + 1;  // keys query 0 sees
  const int keys = min(sp.ctx, first_vis + (min(row0 + ROWS, rows) - 1) / a.group);  // that the tile sees
  const int groups = keys > 0 ? (keys + kGroupKeys - 1) / kGroupKeys : 0;
  const int used = min(splits, max(1, groups / 8));
  if (split >= used) return;
  const int per = (groups + used - 1) / used;
  const int g0 = split * per, g1 = min(groups, g0 + per);

  // Q^T operand: channels 16 s + 8 half .. + 7 of row c
  const int r = row0 + wave * 32 + c;
  const bool on = r < rows;
  const int vis = on ? min(sp.ctx, first_vis + r / a.group) : 0;
  const int wfull = first_vis + (row0 + wave * 32) / a.group;  // keys that all of the wave's rows see
  f16x8_t qf[KSTEP];
  float qmul;
  {
    const int t = sp.q0 + (on ? r / a.group : 0), head = h * a.group + (on ? r % a.group : 0);
    const int64_t at = (int64_t)t * a.qs_t + (int64_t)head * a.qs_h;
    u32x4_t raw[KSTEP];
#pragma unroll
    for (int s = 0; s < KSTEP; ++s) raw[s] = *(const u32x4_t*)((const uint16_t*)a.q + at + 16 * s + 8 * half);
    float x[KSTEP][8], amax = 0.0f;
#pragma unroll
    for (int s = 0; s < KSTEP; ++s) {
      halves_to_f32(raw[s], a.q_f16, x[s]);
#pragma unroll
      for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(x[s][j]));
    }
    const float f = q_factor(half_max(amax));
    qmul = (fabsf(a.scale) * kLog2e) * (1.0f / f);
    const float qf_mul = a.scale < 0.0f ? -f : f;  // the factor of the scores is positive: their maximum is the raw one's
#pragma unroll
    for (int s = 0; s < KSTEP; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) qf[s][j] = (f16_t)(x[s][j] * qf_mul);
  }

  f32x16_t o[DT], sa[2], sb[2];
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = f32x16_t{};
  float mx = kNegInf, l = 0.0f;

  const int32_t* row_table = a.tables + (int64_t)b * a.bt_b;
  const uint8_t* kbase = a.kc + (int64_t)h * a.kc_h;
  const uint8_t* vbase = a.vc + (int64_t)h * a.vc_h;
  const int bmask = (1 << a.shift) - 1;

  // A step's four tiles are looked up by lane: lane i holds tile i % 4.  Ids and
  // scales are kept as loaded until the step that needs them: looking at one
  // earlier would wait for its load.
  const int quad16 = 16 * (lane & 3);
  auto raw_ids = [&](int gi) { return row_table[min(gi * kGroupKeys + quad16, keys - 1) >> a.shift]; };
  auto checked = [&](int gi, int id) {  // -1: no such block, or past the keys
    return ((gi < g1) & (gi * kGroupKeys + quad16 < keys) & (id < a.num_blocks)) ? id : -1;
  };
  auto scale_of = [&](const float* scales, int id) { return scales[(int64_t)max(id, 0) * a.sc_b + h]; };
  auto load_codes = [&](u32x4_t* raw, const uint8_t* base, int64_t stride, int gi, int ids) {
    const int id = max(__builtin_amdgcn_readlane(ids, wave), 0);
    const uint8_t* p = base + (int64_t)id * stride + ((gi * kGroupKeys + 16 * wave) & bmask) * D + lane * 16;
#pragma unroll
    for (int i = 0; i < KP; ++i) raw[i] = *(const u32x4_t*)(p + 1024 * i);
  };
  // the factor of the wave's tile: its scale over the largest so far
  auto factor = [&](float scale, float top) {
    const float s = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, scale), wave));
    const f16_t f = (f16_t)(s * __builtin_amdgcn_rcpf(top));
    return f16x2_t{f, f};
  };
  // Where the lane's first piece goes: chunk 2 p of its row, and 2 p + 1 at ^ 16
  // (the second piece: eight K rows or 64 V rows on, at the same p).
  const uint32_t kw0 = (16 * wave + lane / (D / 16)) * (2 * D) +
                       (((2 * (lane % (D / 16))) ^ lds_swizzle<2 * D>(16 * wave + lane / (D / 16))) << 4);
  const uint32_t vw0 = 2 * KB + lane * 128 + (((2 * wave) ^ lds_swizzle<128>(lane)) << 4);
  auto kw = [&](int i) { return i ? (kw0 + 8 * 2 * D) ^ (8u << 4) : kw0; };
  auto vw = [&](int i) { return vw0 + i * 64 * 128; };
  // One of the 4 KP words of the wave's codes, to halves in w; each second word completes a 16-byte chunk.
  auto convert_k = [&](const u32x4_t* raw, int n, int buf, f16x2_t f, u32x4_t& w) {
    const int i = n >> 2, j = n & 3;
    const u32x2_t x = codes_scaled<FP8>(raw[i][j], f);
    w[2 * (j & 1)] = x[0];
    w[2 * (j & 1) + 1] = x[1];
    if (j & 1) *(u32x4_t*)(s_kv + ((kw(i) ^ (16u * (j >> 1))) + buf * KB)) = w;
  };
  auto convert_v = [&](const u32x4_t* raw, int n, int buf, f16x2_t f, u32x4_t& w) {
    const int i = n >> 2, j = n & 3;  // words 0, 2, then 1, 3
    const u32x2_t x = codes_scaled<FP8>(raw[i][(j >> 1) | ((j & 1) << 1)], f);
    w[2 * (j & 1)] = x[0];
    w[2 * (j & 1) + 1] = x[1];
    if (j & 1) *(u32x4_t*)(s_kv + ((vw(i) ^ (16u * (j >> 1))) + buf * KB)) = w;
  };
  auto drop_past_keys = [&](u32x4_t* raw, int gi, int ids) {
    if constexpr (FP8) {  // V's tokens past the keys may hold NaN codes, and 0 * NaN is no 0
      const int live = __builtin_amdgcn_readlane(ids, wave) < 0 ? 0 : keys - (gi * kGroupKeys + 16 * wave);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int nb = min(max(live - 4 * j, 0), 4);
        const uint32_t keep = (uint32_t)((1ull << (8 * nb)) - 1);
#pragma unroll
        for (int i = 0; i < KP; ++i) raw[i][j] &= keep;
      }
    }
  };
  // the lane's first operand chunks; those of channel step s and of 16 keys u are at ^ 32 s and ^ 32 u
  const uint32_t ka0 = c * (2 * D) + ((half ^ lds_swizzle<2 * D>(c)) << 4);
  const uint32_t va0 = 2 * KB + c * 128 + ((half ^ lds_swizzle<128>(c)) << 4);

  auto mask = [&](f32x16_t(&sx)[2], int gi, unsigned there) {
    const int rel = vis - gi * kGroupKeys - 4 * half;  // keys the row sees of the step, less the lane's first
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int lim = (there >> (2 * x + (j >> 3))) & 1 ? rel : -64;
        sx[x][j] = 32 * x + 8 * (j >> 2) + (j & 3) >= lim ? kNegInf : sx[x][j];
      }
  };
  auto row_max = [&](const f32x16_t(&sx)[2]) {
    float m0 = kNegInf, m1 = kNegInf;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      m0 = fmaxf(fmaxf(m0, sx[0][j]), sx[1][j]);
      ++j;
      m1 = fmaxf(fmaxf(m1, sx[0][j]), sx[1][j]);
    }
    return fmaxf(m0, m1);
  };
  // the running maximum takes in a step's scores (times mul); exp2(fma(score, mul, -base)) are then its weights
  float mul = 0.0f, base = 0.0f;
  auto raise = [&](f32x16_t(&sx)[2], float lane_max, float top_scale) {
    mul = fmaxf(qmul * top_scale, 1e-37f);  // above 0: -inf stays -inf
    const float top = half_max(lane_max) * mul;
    if (__any(top > mx + kLazyMax)) {
      const float mnew = fmaxf(mx, top);
      const float alpha = __builtin_amdgcn_exp2f(mx - (mnew == kNegInf ? 0.0f : mnew));
      mx = mnew;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= alpha;
    }
    base = mx == kNegInf ? 0.0f : mx;
    // scores so large that the product's rounding, which mx has and the fma has not, would show
    if (__builtin_expect(__any(fabsf(base) > 65536.0f), 0)) {
#pragma clang fp contract(off)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float prod = sx[x][j] * mul;
          sx[x][j] = prod - base;
        }
      mul = 1.0f;
      base = 0.0f;
    }
  };
  // weights n and n + 1 of the lane's 32, as halves and in the row's sum
  auto weigh = [&](const f32x16_t(&sx)[2], int n, f16x8_t(&pf)[4]) {
    const int x = n >> 4, j = n & 15;
    f32x2_t p;
    p[0] = __builtin_amdgcn_exp2f(__builtin_fmaf(sx[x][j], mul, -base));
    p[1] = __builtin_amdgcn_exp2f(__builtin_fmaf(sx[x][j + 1], mul, -base));
    const f16x2_t ph = __builtin_convertvector(p, f16x2_t), one = {(f16_t)1.0f, (f16_t)1.0f};
    l = __builtin_amdgcn_fdot2(ph, one, l, false);
    pf[n >> 3][n & 7] = ph[0];
    pf[n >> 3][(n & 7) + 1] = ph[1];
  };
  // operand i of a step's products: K's (channel step i / 2, key half i % 2), then V's (16 keys u, channels 32 d)
  auto operand = [&](int i, int kbuf, int vbuf) {
    const int n = i - 2 * KSTEP;
    const uint32_t at = i < 2 * KSTEP ? kbuf * KB + (i & 1) * (64 * D) + (ka0 ^ (32u * (i >> 1)))
                                      : vbuf * KB + (n % DT) * 4096 + (va0 ^ (32u * (n / DT)));
    return *(const f16x8_t*)(s_kv + at);
  };

  // State at step gi (buffer B = parity): cur its masked scores; kr / vr the codes of K(gi + 2) and V(gi + 1), idk / idv and skr / svr
  // their blocks and scales as loaded; ids3 the ids of gi + 3, not checked.
  u32x4_t kr[KP], vr[KP];
  float ktop = 1.17549435e-38f, vtop = 1.17549435e-38f;  // largest scales of K(gi + 1), V(gi)
  float skr = 0.0f, svr = 0.0f;
  int idk = -1, idv = -1, ids3 = -1;
  auto there_only = [&](float s, int id) { return id < 0 ? 0.0f : s; };
  if (g0 < g1) {
    const int i0 = raw_ids(g0), i1 = raw_ids(g0 + 1), i2 = raw_ids(g0 + 2);
    ids3 = raw_ids(g0 + 3);
    const int id0 = checked(g0, i0), id1 = checked(g0 + 1, i1);
    idk = checked(g0 + 2, i2);
    idv = id1;
    u32x4_t k0[KP], k1[KP], v0[KP];
    load_codes(k0, kbase, a.kc_b, g0, id0);
    load_codes(v0, vbase, a.vc_b, g0, id0);
    load_codes(k1, kbase, a.kc_b, g0 + 1, id1);
    const float sk0 = there_only(scale_of(a.k_scale, id0), id0), sk1 = there_only(scale_of(a.k_scale, id1), id1);
    const float sv0 = there_only(scale_of(a.v_scale, id0), id0);
    load_codes(kr, kbase, a.kc_b, g0 + 2, idk);
    load_codes(vr, vbase, a.vc_b, g0 + 1, idv);
    skr = scale_of(a.k_scale, idk);
    svr = scale_of(a.v_scale, idv);
    const float ktop0 = scalar_max(ktop, quad_max(sk0));
    ktop = scalar_max(ktop0, quad_max(sk1));
    vtop = scalar_max(vtop, quad_max(sv0));
    drop_past_keys(v0, g0, id0);
    const f16x2_t fk0 = factor(sk0, ktop0), fk1 = factor(sk1, ktop), fv0 = factor(sv0, vtop);
    u32x4_t w0, w1, w2;
#pragma unroll
    for (int n = 0; n < 4 * KP; ++n) {
      convert_k(k0, n, 0, fk0, w0);
      convert_k(k1, n, 1, fk1, w1);
      convert_v(v0, n, 0, fv0, w2);
    }
    __syncthreads();
    sa[0] = sa[1] = f32x16_t{};
#pragma unroll
    for (int i = 0; i < 2 * KSTEP; ++i)
      sa[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(operand(i, 0, 0), qf[i >> 1], sa[i & 1], 0, 0, 0);
    const unsigned there = (unsigned)__ballot(id0 >= 0) & 15u;
    if (there != 15u || (g0 + 1) * kGroupKeys > wfull) mask(sa, g0, there);
    raise(sa, row_max(sa), ktop0);
  }
  __syncthreads();  // K(g0) has been read: its buffer takes K(g0 + 2)
  auto step = [&](int gi, auto parity, f32x16_t(&cur)[2], f32x16_t(&nxt)[2]) {
    constexpr int B = decltype(parity)::value;
    // In this order, which the compiler left to itself does not find: operands
    // read AHEAD products before theirs, between the products of the first half
    // the exponentials, between those of the second the codes and the maximum.
    constexpr int NK = 2 * KSTEP, N = NK + 4 * DT, AHEAD = D == 128 ? 2 : 4;
    f16x8_t pf[4], fr[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) fr[i] = operand(i, 1 - B, B);
    nxt[0] = nxt[1] = f32x16_t{};
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      nxt[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fr[i % AHEAD], qf[i >> 1], nxt[i & 1], 0, 0, 0);
      fr[i % AHEAD] = operand(i + AHEAD, 1 - B, B);
#pragma unroll
      for (int n = 0; n < 32 / NK; n += 2) weigh(cur, i * (32 / NK) + n, pf);
      __builtin_amdgcn_sched_barrier(0);
    }
    // K(gi + 2) and V(gi + 1) go into the buffers that step gi - 1 read
    const float sk = there_only(skr, idk), sv = there_only(svr, idv);
    const float ktop2 = scalar_max(ktop, quad_max(sk)), vtop1 = scalar_max(vtop, quad_max(sv));
    const f16x2_t fk = factor(sk, ktop2), fv = factor(sv, vtop1);
    const unsigned there = (unsigned)__ballot(idv >= 0) & 15u;  // of step gi + 1
    drop_past_keys(vr, gi + 1, idv);
    u32x4_t wk, wv;
    float m0 = kNegInf, m1 = kNegInf;
#pragma unroll
    for (int i = 0; i < N - NK; ++i) {
      const int d = i % DT, u = i / DT;
      o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fr[(NK + i) % AHEAD], pf[u], o[d], 0, 0, 0);
      if (NK + i + AHEAD < N) fr[(NK + i) % AHEAD] = operand(NK + i + AHEAD, 1 - B, B);
      constexpr int UNITS = 8 * KP / (N - NK);  // 8 KP words of codes over 4 DT products
      static_assert(UNITS == 1, "one word per product");
      if (i < 4 * KP) convert_k(kr, i, B, fk, wk);
      else convert_v(vr, i - 4 * KP, 1 - B, fv, wv);
#pragma unroll
      for (int n = 0; n < 16 / (N - NK); ++n) {
        const int j = i * (16 / (N - NK)) + n;
        float& m = j & 1 ? m1 : m0;
        m = fmaxf(fmaxf(m, nxt[0][j]), nxt[1][j]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    idv = idk;
    idk = checked(gi + 3, ids3);
    load_codes(kr, kbase, a.kc_b, gi + 3, idk);
    load_codes(vr, vbase, a.vc_b, gi + 2, idv);
    skr = scale_of(a.k_scale, idk);
    svr = scale_of(a.v_scale, idv);
    ids3 = raw_ids(gi + 4);
    float lane_max = fmaxf(m0, m1);
    if (there != 15u || (gi + 2) * kGroupKeys > wfull) {
      mask(nxt, gi + 1, there);
      lane_max = row_max(nxt);
    }
    raise(nxt, lane_max, ktop);
    if (vtop1 > vtop) {
      const float f = vtop * __builtin_amdgcn_rcpf(vtop1);
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= f;
    }
    ktop = ktop2;
    vtop = vtop1;
    __syncthreads();
  };
  const std::integral_constant<int, 0> even{};
  const std::integral_constant<int, 1> odd{};
  for (int gi = g0; gi < g1; gi += 2) {
    step(gi, even, sa, sb);
    if (gi + 1 < g1) step(gi + 1, odd, sb, sa);
  }

  const float sum = half_sum(l);
  // the lane's row again, from a thread id the compiler cannot tell is the same: held over the loop it
  // would cost registers there
  int tid_out = threadIdx.x;
  asm volatile("" : "+v"(tid_out));
  const int r_out = row0 + (tid_out >> 6) * 32 + (tid_out & 31);
  if (r_out >= rows) return;
  const int t = sp.q0 + r_out / a.group, head = h * a.group + r_out % a.group;
  const float inv = used > 1 ? vtop : (sum == 0.0f ? 0.0f : vtop / sum);  // a row that sees no key: zeros
  const int64_t at = part_row(a, split, t, head);
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int ch = 32 * d + 8 * j + 4 * half;
      const f32x4_t v = f32x4_t{o[d][4 * j], o[d][4 * j + 1], o[d][4 * j + 2], o[d][4 * j + 3]} * inv;
      if (used > 1) *(f32x4_t*)(a.part_o + at * D + ch) = v;
      else store_out4(a.out, (int64_t)t * a.os_t + (int64_t)head * a.os_h + ch, v, a.q_f16);
    }
  if (half == 0) {
    if (used > 1) {
      a.part_ml[2 * at] = mx;
      a.part_ml[2 * at + 1] = sum;
    }
    if (a.part_used && split == 0) a.part_used[part_row(a, 0, t, head)] = used;
  }
}

// Joins the parts of the first kernel's rows, a workgroup per (sequence, query,
// head): D / 4 lanes hold a split's part, 1024 / D splits at a time, and meet in
// LDS.  The parts' loads do not wait for the maxima that weigh them.
template <int D>
__global__ __launch_bounds__(256) void block_attn_join_few_kernel(const BlockAttnArgs a, int splits, int share) {
  constexpr int LPR = D / 4, SIDE = 256 / LPR;
  __shared__ f32x4_t s_v[SIDE][LPR];
  __shared__ float s_f[kMaxSplits];
  const unsigned heads = a.num_kv_heads * a.group;
  const int head = blockIdx.x % heads, i = (blockIdx.x / heads) % a.few_rows, b = blockIdx.x / heads / a.few_rows;
  const SeqSpan sp = seq_span(a, b);
  if (i >= sp.n || sp.n > a.few_rows) return;
  const int used = splits_used((sp.ctx + kGroupKeys - 1) / kGroupKeys, splits, share);
  if (used == 1) return;
  const int tid = threadIdx.x, lane = tid & 63, side = tid / LPR, d = (tid % LPR) * 4;
  const f32x4_t none = {0.0f, 0.0f, 0.0f, 0.0f};
  const int64_t row = few_row(a, 0, b, i, head), step = few_row(a, 1, 0, 0, 0);
  f32x4_t p0 = none, p1 = none;
  if (side < used) p0 = *(const f32x4_t*)(a.few_o + (row + side * step) * D + d);
  if (side + SIDE < used) p1 = *(const f32x4_t*)(a.few_o + (row + (side + SIDE) * step) * D + d);
  float top = kNegInf, sum = 0.0f;
  for (int s = lane; s < used; s += 64) top = fmaxf(top, a.few_ml[2 * (row + s * step)]);  // every wave by itself
  top = wave_max(top);
  const float base = top == kNegInf ? 0.0f : top;
  for (int s = lane; s < used; s += 64) {
    const float f = __builtin_amdgcn_exp2f(a.few_ml[2 * (row + s * step)] - base);
    sum += a.few_ml[2 * (row + s * step) + 1] * f;
    if (tid < 64) s_f[s] = f;
  }
  sum = wave_sum(sum);
  __syncthreads();
  f32x4_t v = none;
  if (side < used) v = p0 * s_f[side];
  if (side + SIDE < used) v += p1 * s_f[side + SIDE];
  for (int s = side + 2 * SIDE; s < used; s += SIDE) v += *(const f32x4_t*)(a.few_o + (row + s * step) * D + d) * s_f[s];
  s_v[side][tid % LPR] = v;
  __syncthreads();
  if (tid >= LPR) return;
  for (int k = 1; k < SIDE; ++k) v += s_v[k][tid];
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  store_out4(a.out, (int64_t)(sp.q0 + i) * a.os_t + (int64_t)head * a.os_h + d, v * inv, a.q_f16);
}

// Joins the parts of the second kernel's rows: many rows of few splits, D / 4
// lanes a row, one split after another.
template <int D>
__global__ __launch_bounds__(256) void block_attn_join_kernel(const BlockAttnArgs a, int splits) {
  constexpr int LPR = D / 4, ROWS = 256 / LPR;
  const int heads = a.num_kv_heads * a.group;
  const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / LPR;
  const int t = (int)(row / heads), head = (int)(row % heads), d = (threadIdx.x % LPR) * 4;
  if (t >= a.total_rows) return;
  if (a.cu && (t < a.cu[0] || t >= a.cu[a.num_seqs])) return;  // no sequence's row
  const int used = min(a.part_used[row], splits);
  if (used <= 1) return;
  const int64_t step = (int64_t)a.total_rows * heads;
  float top = kNegInf, sum = 0.0f;
  for (int s = 0; s < used; ++s) top = fmaxf(top, a.part_ml[2 * (row + s * step)]);
  const float base = top == kNegInf ? 0.0f : top;
  f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s = 0; s < used; ++s) {
    const float f = __builtin_amdgcn_exp2f(a.part_ml[2 * (row + s * step)] - base);
    sum += a.part_ml[2 * (row + s * step) + 1] * f;
    v += *(const f32x4_t*)(a.part_o + (row + s * step) * D + d) * f;
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  store_out4(a.out, (int64_t)t * a.os_t + (int64_t)head * a.os_h + d, v * inv, a.q_f16);
}

}  // namespace fdms

using namespace fdms;

template <int D, bool FP8>
static int launch_block_attn(BlockAttnArgs a, int max_seqlen, int few_splits, int few_share, int tile_splits,
                             hipStream_t st) {
  const int64_t pairs = (int64_t)a.num_seqs * a.num_kv_heads, max_rows = (int64_t)max_seqlen * a.group;
  const int64_t heads = (int64_t)a.num_kv_heads * a.group;
  if (few_splits) {
    const dim3 grid((unsigned)(pairs * few_splits));
    if (a.few_rows * a.group <= 16) block_attn_kernel<D, FP8, 1><<<grid, 256, 0, st>>>(a, few_splits, few_share);
    else block_attn_kernel<D, FP8, 2><<<grid, 256, 0, st>>>(a, few_splits, few_share);
    FDMS_LAUNCH_CHECK();
    if (few_splits > 1) {
      const dim3 rows((unsigned)(a.num_seqs * a.few_rows * heads));
      block_attn_join_few_kernel<D><<<rows, 256, 0, st>>>(a, few_splits, few_share);
      FDMS_LAUNCH_CHECK();
    }
  }
  if (tile_splits) {
    const dim3 grid((unsigned)(pairs * tile_splits), (unsigned)((max_rows - 1) / kTileRows + 1));
    block_attn_tile_kernel<D, FP8><<<grid, 64 * kTileWaves, 0, st>>>(a, tile_splits);
    FDMS_LAUNCH_CHECK();
    if (tile_splits > 1) {
      constexpr int kPer = 256 / (D / 4);
      block_attn_join_kernel<D><<<dim3((unsigned)((a.total_rows * heads - 1) / kPer + 1)), 256, 0, st>>>(a, tile_splits);
      FDMS_LAUNCH_CHECK();
    }
  }
  return 0;
}

FDMS_EXPORT int fdms_block_attention(const void* q, int q_dtype, int64_t qs_t, int64_t qs_h, int total_rows,
                                     const void* k_cache, const void* v_cache, int is_fp8, int64_t kc_b, int64_t kc_h,
                                     int64_t vc_b, int64_t vc_h, const float* k_scale, const float* v_scale,
                                     int64_t sc_b, const int32_t* block_tables, int64_t bt_b, int width,
                                     const int32_t* context_lens, const int32_t* cu_seqlens, void* out, int64_t os_t,
                                     int64_t os_h, float* workspace, int num_seqs, int num_kv_heads, int group_size,
                                     int head_dim, int num_blocks, int block_size, int max_seqlen, int few_rows,
                                     int few_splits, int few_share, int tile_splits, float scale, void* stream) {
  if ((q_dtype != kF16 && q_dtype != kBF16) || total_rows < 0 || num_seqs < 1 || num_kv_heads < 1 || group_size < 1 ||
      (head_dim != 64 && head_dim != 128) || max_seqlen < 1 || width < 0 || num_blocks < 1 || block_size < 16 ||
      block_size > 256 || (block_size & (block_size - 1)) ||
      (cu_seqlens == nullptr && (max_seqlen != 1 || total_rows != num_seqs)) || !std::isfinite(scale))
    return (int)hipErrorInvalidValue;
  // every sequence length has its kernel: up to few_rows query rows the one, past them the other
  const int splits = few_splits > tile_splits ? few_splits : tile_splits;
  if (few_rows < 0 || (int64_t)few_rows * group_size > 32 || few_splits < 0 || tile_splits < 0 || splits < 1 ||
      splits > kMaxSplits || few_share < 1 || (few_rows > 0 && few_splits == 0) || (few_rows < max_seqlen && tile_splits == 0) ||
      (splits > 1 && workspace == nullptr))
    return (int)hipErrorInvalidValue;
  if (!fdms_aligned16(q, k_cache, v_cache, workspace) || (uintptr_t)out % 8 || qs_t % 8 || qs_h % 8 || os_t % 4 ||
      os_h % 4 || kc_b % 16 || kc_h % 16 || vc_b % 16 || vc_h % 16)
    return (int)hipErrorInvalidValue;
  const int64_t pairs = (int64_t)num_seqs * num_kv_heads, max_rows = (int64_t)max_seqlen * group_size;
  const int64_t heads = (int64_t)num_kv_heads * group_size, rows = total_rows * heads;
  if (pairs * splits > 0x7FFFFFFF || (max_rows - 1) / kTileRows + 1 > 65535 || max_rows > 0x7FFFFFFF ||
      rows > 0x7FFFFFFF ||
      heads * num_seqs * few_rows > 0x7FFFFFFF)
    return (int)hipErrorInvalidValue;
  if (total_rows == 0) return 0;
  BlockAttnArgs a;
  a.q = q, a.qs_t = qs_t, a.qs_h = qs_h;
  a.out = out, a.os_t = os_t, a.os_h = os_h;
  a.kc = (const uint8_t*)k_cache, a.kc_b = kc_b, a.kc_h = kc_h;
  a.vc = (const uint8_t*)v_cache, a.vc_b = vc_b, a.vc_h = vc_h;
  a.k_scale = k_scale, a.v_scale = v_scale, a.sc_b = sc_b;
  a.tables = block_tables, a.bt_b = bt_b, a.width = width;
  a.context = context_lens, a.cu = cu_seqlens;
  // (a count of 1 writes no parts)
  const int64_t few_parts = few_splits > 1 ? few_splits * heads * num_seqs * few_rows : 0;
  const int64_t tile_parts = tile_splits > 1 ? tile_splits * rows : 0;
  a.few_o = workspace;
  a.part_o = a.few_o + few_parts * head_dim;
  a.few_ml = a.part_o + tile_parts * head_dim;
  a.part_ml = a.few_ml + few_parts * 2;
  a.part_used = tile_splits > 1 ? (int*)(a.part_ml + tile_parts * 2) : nullptr;
  a.num_blocks = num_blocks, a.shift = __builtin_ctz(block_size), a.num_seqs = num_seqs;
  a.num_kv_heads = num_kv_heads, a.group = group_size, a.total_rows = total_rows;
  a.few_rows = few_rows, a.q_f16 = q_dtype == kF16, a.scale = scale;
  hipStream_t st = (hipStream_t)stream;
#define FDMS_ATTN(D, F) return launch_block_attn<D, F>(a, max_seqlen, few_splits, few_share, tile_splits, st)
  if (head_dim == 64) {
    if (is_fp8) FDMS_ATTN(64, true);
    FDMS_ATTN(64, false);
  }
  if (is_fp8) FDMS_ATTN(128, true);
  FDMS_ATTN(128, false);
#undef FDMS_ATTN
}
