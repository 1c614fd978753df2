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
#include "fdms_block_kv.h"

namespace fdms {

constexpr int kGroupKeys = 64;  // keys a wave takes at once: four tiles
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
  float* part_o;      // [pair][tile][split][rows][D]
  float* part_ml;     // [pair][tile][split][rows][2]
  int width, num_blocks, shift, num_seqs, num_kv_heads, group, total_rows, splits, tiles;
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

// The splits a query tile uses of the launch's: at least four 64-key groups
// each (one per wave), so a short context leaves the rest of its workgroups idle.
__device__ __forceinline__ int splits_used(int groups, int splits) {
  return min(splits, max(1, (groups + 3) >> 2));
}

__device__ __forceinline__ void store_out4(void* out, int64_t at, f32x4_t v, int f16) {
  u32x2_t r;
  if (f16) {
    const f16x4_t h = __builtin_convertvector(v, f16x4_t);
    r = __builtin_bit_cast(u32x2_t, h);
  } else {
    r[0] = f32_to_bf16(v[0]) | (f32_to_bf16(v[1]) << 16);
    r[1] = f32_to_bf16(v[2]) | (f32_to_bf16(v[3]) << 16);
  }
  *(u32x2_t*)((uint16_t*)out + at) = r;
}

// Power of two that brings a row of largest magnitude amax near 2^14, so the
// row's bf16 values are halves exactly down to 2^-31 of the largest.  Rows of
// zeros, infinities or NaN are left as they are.
__device__ __forceinline__ float q_factor(float amax) {
  const int e = (int)(__float_as_uint(amax) >> 23) - 127;
  if (!(amax > 0.0f) || e > 127) return 1.0f;
  return __uint_as_float((uint32_t)(min(14 - e, 126) + 127) << 23);
}

// One workgroup: 16 * MT query rows (row r: token r / group, head r % group of
// the kv head) of a sequence over one split of its keys; its four waves take
// 64-key groups in turn and join at the end.
template <int D, bool FP8, int MT>
__global__ __launch_bounds__(256) void block_attn_kernel(const BlockAttnArgs a) {
  constexpr int KL = D / 64, DC = D / 16, KS = D / 32;  // K loads per row and lane, V row groups, K steps
  constexpr int ROWS = 16 * MT, PAD = D + 4;
  __shared__ float s_o[4][ROWS][PAD];
  __shared__ float s_ml[4][ROWS][2];
  const int pairs = a.num_seqs * a.num_kv_heads;
  const int pair = blockIdx.x % pairs, split = blockIdx.x / pairs, tile = blockIdx.y;
  const int b = pair / a.num_kv_heads, h = pair % a.num_kv_heads;
  const SeqSpan sp = seq_span(a, b);
  const int rows = sp.n * a.group, row0 = tile * ROWS;
  if (sp.n <= 0 || row0 >= rows) return;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, c = lane & 15;
  const int first_vis = sp.ctx - sp.n + 1;  // keys query 0 sees
  const int last_row = min(row0 + ROWS, rows) - 1;
  const int keys = min(sp.ctx, first_vis + last_row / a.group);  // keys the tile sees (may be <= 0)
  const int full = first_vis + row0 / a.group;                   // keys that all of its rows see
  const int groups = keys > 0 ? (keys + kGroupKeys - 1) / kGroupKeys : 0;
  const int used = splits_used(groups, a.splits);
  if (split >= used) return;
  const int per = (groups + used - 1) / used;
  const int g_end = min(groups, (split + 1) * per);

  // Q^T operand: lane (g, c) holds channels a * 64 + g * 16 + 8 * half .. + 7 of row c
  f16x8_t qf[MT][KS];
  float qmul[MT];  // score factor of the lane's row
  int vis[MT];     // keys it sees
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int r = row0 + m * 16 + c;
    const bool on = r < rows;
    const int i = on ? r / a.group : 0, hq = h * a.group + (on ? r % a.group : 0);
    vis[m] = on ? min(sp.ctx, first_vis + i) : 0;
    const int64_t at = (int64_t)(sp.q0 + i) * a.qs_t + (int64_t)hq * a.qs_h;
    float x[KS][8], amax = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const u32x4_t raw = *(const u32x4_t*)((const uint16_t*)a.q + at + (s >> 1) * 64 + g * 16 + (s & 1) * 8);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t e = (raw[j >> 1] >> (16 * (j & 1))) & 0xFFFFu;
        x[s][j] = a.q_f16 ? (float)__builtin_bit_cast(f16_t, (uint16_t)e) : bf16_to_f32(e);
        amax = fmaxf(amax, fabsf(x[s][j]));
      }
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

  for (int gi = split * per + wave; gi < g_end; gi += 4) {
    const int key0 = gi * kGroupKeys;
    // the lane's V tile (g) and the tile of its K rows (c / 4)
    const int kv_v = key0 + 16 * g, kv_k = key0 + 16 * (c >> 2);
    const int idv = kv_v < keys ? row_table[kv_v >> a.shift] : -1;
    const int idk = kv_k < keys ? row_table[kv_k >> a.shift] : -1;
    const bool okv = idv >= 0 && idv < a.num_blocks, okk = idk >= 0 && idk < a.num_blocks;
    const uint8_t* kp = kbase + (int64_t)(okk ? idk : 0) * a.kc_b + ((kv_k & bmask) + (c & 3)) * D + g * 16;
    const uint8_t* vp = vbase + (int64_t)(okv ? idv : 0) * a.vc_b + (kv_v & bmask) * D + c * kTile;
    u32x4_t kr[4][KL], vr[DC];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int x = 0; x < KL; ++x) kr[t][x] = *(const u32x4_t*)(kp + 4 * t * D + 64 * x);
#pragma unroll
    for (int d = 0; d < DC; ++d) vr[d] = *(const u32x4_t*)(vp + 256 * d);
    const int64_t sc = (int64_t)(okv ? idv : 0) * a.sc_b + h;
    const float sk = okv ? a.k_scale[sc] : 0.0f, sv = okv ? a.v_scale[sc] : 0.0f;
    const int live = okv ? keys - kv_v : 0;  // of the lane's tile; rows past it hold whatever the block held
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
    const float sv_top = rows_max(sv);
    float osc = 1.0f;
    if (sv_top > sref) {
      osc = sref / sv_top;
      sref = sv_top;
    }
    const float vmul = sv / sref;
    const bool masked = __any(!okv) || key0 + kGroupKeys > full;

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
    }
    f16x8_t pf[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const float mul = qmul[m] * sk;
      float top = kNegInf;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float x = st[m][t][r] * mul;
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
#pragma unroll
    for (int d = 0; d < DC; ++d)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const f16x8_t vf = codes8_to_f16<FP8>(vr[d][2 * u], vr[d][2 * u + 1]);
#pragma unroll
        for (int m = 0; m < MT; ++m) o[m][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[m][u], o[m][d], 0, 0, 0);
      }
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
    const int r = e / (D / 4), d = (e % (D / 4)) * 4, row = row0 + r;
    if (row >= rows) break;
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
      store_out4(a.out, (int64_t)(sp.q0 + row / a.group) * a.os_t + (int64_t)(h * a.group + row % a.group) * a.os_h + d,
                 v * inv, a.q_f16);
    } else {
      const int64_t at = (((int64_t)pair * a.tiles + tile) * a.splits + split) * ROWS + r;
      *(f32x4_t*)(a.part_o + at * D + d) = v;
      if (d == 0) {
        a.part_ml[2 * at] = top;
        a.part_ml[2 * at + 1] = sum;
      }
    }
  }
}

// Joins the splits of the rows that used several: D / 4 lanes per row.
template <int D, int ROWS>
__global__ __launch_bounds__(256) void block_attn_join_kernel(const BlockAttnArgs a) {
  constexpr int LPR = D / 4, RPG = 256 / LPR;
  const int pair = blockIdx.x, b = pair / a.num_kv_heads, h = pair % a.num_kv_heads;
  const SeqSpan sp = seq_span(a, b);
  const int rows = sp.n * a.group;
  const int row = blockIdx.y * RPG + threadIdx.x / LPR, d = (threadIdx.x % LPR) * 4;
  if (sp.n <= 0 || row >= rows) return;
  const int tile = row / ROWS, last_row = min((tile + 1) * ROWS, rows) - 1;
  const int keys = min(sp.ctx, sp.ctx - sp.n + 1 + last_row / a.group);
  const int used = splits_used(keys > 0 ? (keys + kGroupKeys - 1) / kGroupKeys : 0, a.splits);
  if (used == 1) return;
  const int64_t at = ((int64_t)pair * a.tiles + tile) * a.splits * ROWS + row % ROWS;
  float top = kNegInf;
  for (int s = 0; s < used; ++s) top = fmaxf(top, a.part_ml[2 * (at + (int64_t)s * ROWS)]);
  const float base = top == kNegInf ? 0.0f : top;
  float sum = 0.0f;
  f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s = 0; s < used; ++s) {
    const int64_t p = at + (int64_t)s * ROWS;
    const float f = __builtin_amdgcn_exp2f(a.part_ml[2 * p] - base);
    sum += a.part_ml[2 * p + 1] * f;
    v += *(const f32x4_t*)(a.part_o + p * D + d) * f;
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  store_out4(a.out, (int64_t)(sp.q0 + row / a.group) * a.os_t + (int64_t)(h * a.group + row % a.group) * a.os_h + d,
             v * inv, a.q_f16);
}

}  // namespace fdms

using namespace fdms;

template <int D, bool FP8, int MT>
static int launch_block_attn(const BlockAttnArgs& a, int max_rows, hipStream_t st) {
  const int64_t pairs = (int64_t)a.num_seqs * a.num_kv_heads;
  block_attn_kernel<D, FP8, MT><<<dim3((unsigned)(pairs * a.splits), a.tiles), 256, 0, st>>>(a);
  FDMS_LAUNCH_CHECK();
  if (a.splits > 1) {
    constexpr int RPG = 256 / (D / 4);
    block_attn_join_kernel<D, 16 * MT><<<dim3((unsigned)pairs, (max_rows - 1) / RPG + 1), 256, 0, st>>>(a);
    FDMS_LAUNCH_CHECK();
  }
  return 0;
}

FDMS_EXPORT int fdms_block_attention(const void* q, int q_dtype, int64_t qs_t, int64_t qs_h, int total_rows,
                                     const void* k_cache, const void* v_cache, int is_fp8, int64_t kc_b, int64_t kc_h,
                                     int64_t vc_b, int64_t vc_h, const float* k_scale, const float* v_scale,
                                     int64_t sc_b, const int32_t* block_tables, int64_t bt_b, int width,
                                     const int32_t* context_lens, const int32_t* cu_seqlens, void* out, int64_t os_t,
                                     int64_t os_h, float* workspace, int num_seqs, int num_kv_heads, int group_size,
                                     int head_dim, int num_blocks, int block_size, int max_seqlen, int tile_rows,
                                     int num_splits, float scale, void* stream) {
  if ((q_dtype != kF16 && q_dtype != kBF16) || total_rows < 0 || num_seqs < 1 || num_kv_heads < 1 || group_size < 1 ||
      (head_dim != 64 && head_dim != 128) || max_seqlen < 1 || width < 0 || num_blocks < 1 || block_size < 16 ||
      block_size > 256 || (block_size & (block_size - 1)) || num_splits < 1 || num_splits > 1024 ||
      (tile_rows != 16 && tile_rows != 32) || (num_splits > 1 && workspace == nullptr) ||
      (cu_seqlens == nullptr && (max_seqlen != 1 || total_rows != num_seqs)))
    return (int)hipErrorInvalidValue;
  if (!fdms_aligned16(q, k_cache, v_cache, workspace) || (uintptr_t)out % 8 || qs_t % 8 || qs_h % 8 || os_t % 4 ||
      os_h % 4 || kc_b % 16 || kc_h % 16 || vc_b % 16 || vc_h % 16)
    return (int)hipErrorInvalidValue;
  const int64_t pairs = (int64_t)num_seqs * num_kv_heads, max_rows = (int64_t)max_seqlen * group_size;
  const int64_t tiles = (max_rows - 1) / tile_rows + 1;
  if (pairs * num_splits > 0x7FFFFFFF || tiles > 65535 || (int64_t)total_rows * group_size > 0x7FFFFFFF)
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
  a.part_o = workspace, a.part_ml = workspace + pairs * tiles * num_splits * tile_rows * head_dim;
  a.num_blocks = num_blocks, a.shift = __builtin_ctz(block_size), a.num_seqs = num_seqs;
  a.num_kv_heads = num_kv_heads, a.group = group_size, a.total_rows = total_rows;
  a.splits = num_splits, a.tiles = (int)tiles, a.q_f16 = q_dtype == kF16, a.scale = scale;
  hipStream_t st = (hipStream_t)stream;
  const int rows = (int)max_rows;
#define FDMS_ATTN(D, F) \
  return tile_rows == 16 ? launch_block_attn<D, F, 1>(a, rows, st) : launch_block_attn<D, F, 2>(a, rows, st)
  if (head_dim == 64) {
    if (is_fp8) FDMS_ATTN(64, true);
    FDMS_ATTN(64, false);
  }
  if (is_fp8) FDMS_ATTN(128, true);
  FDMS_ATTN(128, false);
#undef FDMS_ATTN
}
