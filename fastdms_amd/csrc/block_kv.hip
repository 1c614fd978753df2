// Dense 8-bit block KV cache: block tables and slot maps from request
// lengths, the store of new K/V rows, and the dense read-back of cached rows
// (layout: fdms_block_kv.h).
#include "fdms_block_kv.h"

namespace fdms {

// ------------------------------------------------------------------ block tables
// Sequence b holds cached[b] tokens in ceil(cached / bs) blocks and gets
// fresh[b] more.  With cu the exclusive sums of fresh and first those of the
// new blocks ceil((cached + fresh) / bs) - ceil(cached / bs), token t of
// sequence b is position p = cached[b] + t - cu[b], in block p / bs of the
// sequence's row: a held entry of the table, or the (first[b] + p / bs - held)-th
// block popped from the stack's top.  The token that opens a block writes its
// table entry, so no entry is both read and written.
//
// One launch: every workgroup sums the (at most 4096) lengths itself -- 32 KB
// that sit in the L2 -- and then maps its own tokens by a binary search of cu
// in LDS.  A second launch for the map would cost more than the repeated sums.
constexpr int kTabThreads = 1024;
constexpr int kTabSeqs = 4 * kTabThreads;
constexpr int kTabTokens = 2 * kTabThreads;  // tokens mapped per workgroup

enum : int { kTabNoBlocks = 1, kTabNarrow = 2, kTabTokensShort = 4, kTabInvalid = 8 };

__device__ __forceinline__ int64_t wave_scan_i64(int64_t v) {
  const int lane = lane_id();
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int64_t u = __shfl_up(v, o, kWave);
    if (lane >= o) v += u;
  }
  return v;
}

__global__ __launch_bounds__(kTabThreads) void block_tables_kernel(
    const int32_t* __restrict__ cached, const int32_t* __restrict__ fresh, int num_seqs, int32_t* tables,
    int64_t bt_b, int width, const int32_t* __restrict__ stack, int stack_len, const int32_t* __restrict__ count,
    int shift, int num_tokens, int32_t* __restrict__ slots, int64_t* __restrict__ positions,
    int32_t* __restrict__ cu_out, int32_t* __restrict__ context, int32_t* __restrict__ count_out,
    int32_t* __restrict__ status_out) {
  __shared__ int s_cu[kTabSeqs + 1];
  __shared__ int s_first[kTabSeqs];
  __shared__ int64_t s_wave[2][kTabThreads / kWave];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int bs = 1 << shift;
  const int held_free = *count;
  int bad = (held_free < 0 || held_free > stack_len) ? kTabInvalid : 0;
  int64_t tok[4], blk[4], tsum = 0, bsum = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int b = tid * 4 + j;
    tok[j] = blk[j] = 0;
    if (b < num_seqs) {
      const int64_t c = cached[b], n = fresh[b];
      if (c < 0 || n < 0 || c + n > 0x7FFFFFFF) {
        bad |= kTabInvalid;
      } else {
        const int64_t need = (c + n + bs - 1) >> shift;
        if (need > width) bad |= kTabNarrow;
        tok[j] = n;
        blk[j] = need - ((c + bs - 1) >> shift);
      }
    }
    tsum += tok[j];
    bsum += blk[j];
  }
  const int64_t tinc = wave_scan_i64(tsum), binc = wave_scan_i64(bsum);
  if (lane == kWave - 1) {
    s_wave[0][wave] = tinc;
    s_wave[1][wave] = binc;
  }
  __syncthreads();
  int64_t tbase = tinc - tsum, bbase = binc - bsum, ttotal = 0, btotal = 0;
  for (int w = 0; w < kTabThreads / kWave; ++w) {
    if (w < wave) {
      tbase += s_wave[0][w];
      bbase += s_wave[1][w];
    }
    ttotal += s_wave[0][w];
    btotal += s_wave[1][w];
  }
  if (ttotal > num_tokens) bad |= kTabTokensShort;
  if (btotal > held_free) bad |= kTabNoBlocks;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int b = tid * 4 + j;
    if (b < num_seqs) {
      s_cu[b] = (int)tbase;
      s_first[b] = (int)bbase;
    }
    tbase += tok[j];
    bbase += blk[j];
  }
  if (tid == 0) s_cu[num_seqs] = (int)ttotal;
  // the flags of all threads (the call is also the barrier behind s_cu)
  int status = 0;
  for (int bit = 1; bit <= kTabInvalid; bit <<= 1) status |= __syncthreads_or(bad & bit) ? bit : 0;

  if (blockIdx.x == 0) {
    for (int b = tid; b <= num_seqs; b += kTabThreads) {
      cu_out[b] = status ? 0 : s_cu[b];
      if (b < num_seqs) context[b] = status ? max(cached[b], 0) : cached[b] + fresh[b];
    }
    if (tid == 0) {
      *count_out = status ? held_free : held_free - (int)btotal;
      *status_out = status;
    }
  }
#pragma unroll
  for (int j = 0; j < kTabTokens / kTabThreads; ++j) {
    const int64_t t = (int64_t)blockIdx.x * kTabTokens + j * kTabThreads + tid;
    if (t >= num_tokens) break;
    int64_t slot = -1, p = 0;
    if (status == 0 && t < ttotal) {
      int lo = 0, hi = num_seqs;  // cu[lo] <= t < cu[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_cu[mid] <= t) lo = mid;
        else hi = mid;
      }
      const int c = cached[lo];
      p = c + (t - s_cu[lo]);
      const int at = (int)(p >> shift), held = (c + bs - 1) >> shift, off = (int)p & (bs - 1);
      int32_t* entry = tables + (int64_t)lo * bt_b + at;
      int id;
      if (at < held) {
        id = *entry;
      } else {
        id = stack[held_free - 1 - (s_first[lo] + at - held)];
        if (off == 0) *entry = id;
      }
      const int64_t s = ((int64_t)id << shift) + off;
      if (id >= 0 && s <= 0x7FFFFFFF) slot = s;
    }
    slots[t] = (int)slot;
    positions[t] = p;
  }
}

// ------------------------------------------------------------------ store
// Rows t0 .. t0 + n - 1 with consecutive slots of one block are a run; the
// workgroup whose tokens hold a run's first row stores the whole run, one wave
// per 16-row tile of the block, for one kv head and K or V.  The new rows stay
// in registers between their amax and their codes, so each is read once.  When
// the run raises the block's scale, the rows before it are encoded again.
//
// Bound by HBM: 4 bytes read per value pair and 2 written; a prompt's blocks
// are independent, so the grid covers them all at once.
constexpr int kKPass = 4;  // at most: passes of 64 lanes over a 16-row K tile of 8-channel pieces

template <typename T>
__device__ __forceinline__ void load_row8(const T* p, float* x) {
  if constexpr (sizeof(T) == 2) {
    const u32x4_t r = *(const u32x4_t*)p;
    const T* e = (const T*)&r;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = ld<T>(e + i);
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x4_t r = *(const f32x4_t*)(p + 4 * h);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * h + i] = r[i];
    }
  }
}
template <typename T>
__device__ __forceinline__ void load_pair(const T* p, float* x0, float* x1) {
  if constexpr (sizeof(T) == 2) {
    const uint32_t r = *(const uint32_t*)p;
    const T* e = (const T*)&r;
    *x0 = ld<T>(e);
    *x1 = ld<T>(e + 1);
  } else {
    const f32x2_t r = *(const f32x2_t*)p;
    *x0 = r[0];
    *x1 = r[1];
  }
}

// Max over the workgroup (WAVES waves); every thread calls it.
template <int WAVES>
__device__ __forceinline__ float team_max(float v, float* s_red) {
  v = wave_max(v);
  if constexpr (WAVES > 1) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s_red[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) v = fmaxf(v, s_red[w]);
  }
  return v;
}

// The scale of a block after a run's rows (amax) joined `off` earlier ones.
template <bool FP8>
__device__ __forceinline__ float joined_scale(float amax, int off, float old) {
  const float need = block_scale<FP8>(amax);
  return off > 0 ? fmaxf(old, need) : need;
}

template <typename T, int D, bool FP8, int WAVES>
__device__ __forceinline__ void store_run_k(const T* __restrict__ x, int64_t xs_t, uint8_t* block, float* scale,
                                            int off, int n, float* s_red) {
  constexpr int LPR = D / 8, RPP = kWave / LPR, PASS = kTile / RPP;
  static_assert(PASS <= kKPass, "tile passes");
  const int lane = lane_id(), row0 = (threadIdx.x >> 6) * kTile + lane / LPR, d0 = (lane % LPR) * 8;
  float v[PASS][8], amax = 0.0f;
#pragma unroll
  for (int i = 0; i < PASS; ++i) {
    const int r = row0 + i * RPP;
    if (r >= off && r < off + n) {
      load_row8<T>(x + (int64_t)(r - off) * xs_t + d0, v[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[i][j] = nan_to_zero(v[i][j]);
        amax = fmaxf(amax, fabsf(v[i][j]));
      }
    }
  }
  const float old = *scale, s = joined_scale<FP8>(team_max<WAVES>(amax, s_red), off, old);
  const float inv = 1.0f / s;
  const bool grown = off > 0 && s > old;
  const float ratio = old * inv;
#pragma unroll
  for (int i = 0; i < PASS; ++i) {
    const int r = row0 + i * RPP;
    u32x2_t* dst = (u32x2_t*)(block + r * D + d0);
    if (r >= off && r < off + n) {
      u32x2_t c;
      c[0] = encode4<FP8>(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv);
      c[1] = encode4<FP8>(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv);
      *dst = c;
    } else if (grown && r < off) {
      u32x2_t c = *dst;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t w = c[j];
        c[j] = encode4<FP8>(code_value<FP8>(w, 0) * ratio, code_value<FP8>(w, 1) * ratio,
                            code_value<FP8>(w, 2) * ratio, code_value<FP8>(w, 3) * ratio);
      }
      *dst = c;
    }
  }
  if (threadIdx.x == 0) *scale = s;
}

// V: a lane holds two channels of 16 (D = 128) or 8 (D = 64) tokens of its
// wave's tile, the bytes it stores.
template <typename T, int D, bool FP8, int WAVES>
__device__ __forceinline__ void store_run_v(const T* __restrict__ x, int64_t xs_t, uint8_t* block, float* scale,
                                            int off, int n, float* s_red) {
  constexpr int LPR = D / 2, TOK = kTile * LPR / kWave, WORDS = TOK / 4;
  const int lane = lane_id(), tile = threadIdx.x >> 6, d0 = (lane % LPR) * 2, t0 = (lane / LPR) * TOK;
  const int row0 = tile * kTile + t0;
  float v[2][TOK], amax = 0.0f;
#pragma unroll
  for (int j = 0; j < TOK; ++j) {
    const int r = row0 + j;
    v[0][j] = v[1][j] = 0.0f;
    if (r >= off && r < off + n) {
      load_pair<T>(x + (int64_t)(r - off) * xs_t + d0, &v[0][j], &v[1][j]);
      v[0][j] = nan_to_zero(v[0][j]);
      v[1][j] = nan_to_zero(v[1][j]);
      amax = fmaxf(amax, fmaxf(fabsf(v[0][j]), fabsf(v[1][j])));
    }
  }
  const float old = *scale, s = joined_scale<FP8>(team_max<WAVES>(amax, s_red), off, old);
  const float inv = 1.0f / s;
  const bool grown = off > 0 && s > old;
  const float ratio = old * inv;
  const bool any_new = row0 < off + n && row0 + TOK > off;
  if (any_new || (grown && row0 < off)) {
    const bool whole = row0 >= off && row0 + TOK <= off + n;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      uint32_t* dst = (uint32_t*)(block + (int64_t)tile * (D * kTile) + (d0 + c) * kTile + t0);
#pragma unroll
      for (int w = 0; w < WORDS; ++w) {
        uint32_t code = encode4<FP8>(v[c][4 * w] * inv, v[c][4 * w + 1] * inv, v[c][4 * w + 2] * inv,
                                     v[c][4 * w + 3] * inv);
        if (!whole) {  // bytes of the rows before (encoded again if the scale grew) and of those behind
          const uint32_t was = dst[w];
          uint32_t again = was;
          if (grown)
            again = encode4<FP8>(code_value<FP8>(was, 0) * ratio, code_value<FP8>(was, 1) * ratio,
                                 code_value<FP8>(was, 2) * ratio, code_value<FP8>(was, 3) * ratio);
          uint32_t mixed = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = row0 + 4 * w + j;
            const uint32_t from = r < off ? again : (r < off + n ? code : was);
            mixed |= from & (0xFFu << (8 * j));
          }
          code = mixed;
        }
        dst[w] = code;
      }
    }
  }
  if (threadIdx.x == 0) *scale = s;
}

template <typename T, int D, bool FP8, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void store_block_kernel(
    const T* __restrict__ k, int64_t ks_t, int64_t ks_h, const T* __restrict__ v, int64_t vs_t, int64_t vs_h,
    uint8_t* kc, int64_t kc_b, int64_t kc_h, uint8_t* vc, int64_t vc_b, int64_t vc_h, float* k_scale,
    float* v_scale, int64_t sc_b, const int32_t* __restrict__ slots,
    int num_tokens, int num_blocks, int per_group) {
  constexpr int BS = kTile * WAVES;
  __shared__ float s_red[WAVES];
  const int h = blockIdx.y, lane = lane_id();
  const bool is_v = blockIdx.z != 0;
  int64_t t = (int64_t)blockIdx.x * per_group;
  const int64_t end = min(t + per_group, (int64_t)num_tokens);
  while (t < end) {
    const int slot = slots[t];
    const int blk = slot / BS, off = slot & (BS - 1);
    if (slot < 0 || blk >= num_blocks) {
      ++t;
      continue;
    }
    const bool first = off == 0 || t == 0 || slots[t - 1] != slot - 1;
    int n = 0;  // rows of the run: the leading lanes whose slots follow on
    for (int i0 = 0; i0 < BS; i0 += kWave) {
      const int i = i0 + lane;
      const bool on = off + i < BS && t + i < num_tokens && slots[t + i] == slot + i;
      const uint64_t m = ~__ballot(on);
      const int run = m ? __builtin_ctzll(m) : kWave;
      n += run;
      if (run < kWave) break;
    }
    if (first) {
      if (is_v)
        store_run_v<T, D, FP8, WAVES>(v + t * vs_t + h * vs_h, vs_t, vc + blk * vc_b + h * vc_h,
                                      v_scale + blk * sc_b + h, off, n, s_red);
      else
        store_run_k<T, D, FP8, WAVES>(k + t * ks_t + h * ks_h, ks_t, kc + blk * kc_b + h * kc_h,
                                      k_scale + blk * sc_b + h, off, n, s_red);
    }
    t += n;
  }
}

// ------------------------------------------------------------------ read-back
// Dense rows of the tokens at slots[t]; a slot outside the cache gives zeros.
// A wave takes 16 tokens of one kv head, K or V.  V comes from transposed
// tiles: a lane keeps the 16 tokens of its two channels in registers while the
// tokens stay in one tile, so a run of slots reads each tile once.
template <typename TO, int D, bool FP8>
__global__ __launch_bounds__(256) void gather_block_kernel(
    const uint8_t* __restrict__ kc, int64_t kc_b, int64_t kc_h, const uint8_t* __restrict__ vc, int64_t vc_b,
    int64_t vc_h, const float* __restrict__ k_scale, const float* __restrict__ v_scale, int64_t sc_b,
    const int32_t* __restrict__ slots, int num_tokens, int num_blocks, int shift, TO* __restrict__ out_k,
    int64_t ok_t, int64_t ok_h, TO* __restrict__ out_v, int64_t ov_t, int64_t ov_h) {
  constexpr int LPR = D / 2, TOK = kTile * LPR / kWave;  // lanes per row, tokens per lane
  const int h = blockIdx.y, lane = lane_id();
  const bool is_v = blockIdx.z != 0;
  const int64_t t0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * kTile + (lane / LPR) * TOK;
  const int d0 = (lane % LPR) * 2;
  const int mask = (1 << shift) - 1;
  TO* out = is_v ? out_v : out_k;
  const int64_t os_t = is_v ? ov_t : ok_t, os_h = is_v ? ov_h : ok_h;
  int tile = -1;
  u32x4_t c0 = {0, 0, 0, 0}, c1 = {0, 0, 0, 0};
  float s = 0.0f;
#pragma unroll 4
  for (int i = 0; i < TOK; ++i) {
    const int64_t t = t0 + i;
    if (t >= num_tokens) break;
    const int slot = slots[t];
    const int blk = slot >> shift, off = slot & mask;
    float x0 = 0.0f, x1 = 0.0f;
    if (slot >= 0 && blk < num_blocks) {
      if (is_v) {
        if (slot >> 4 != tile) {
          tile = slot >> 4;
          const u32x4_t* p = (const u32x4_t*)(vc + blk * vc_b + h * vc_h + (off >> 4) * (D * kTile) + d0 * kTile);
          c0 = p[0];
          c1 = p[1];
          s = v_scale[blk * sc_b + h];
        }
        const int w = (off >> 2) & 3;
        const uint32_t a = w == 0 ? c0[0] : w == 1 ? c0[1] : w == 2 ? c0[2] : c0[3];
        const uint32_t b = w == 0 ? c1[0] : w == 1 ? c1[1] : w == 2 ? c1[2] : c1[3];
        x0 = code_value<FP8>(a, off & 3) * s;
        x1 = code_value<FP8>(b, off & 3) * s;
      } else {
        const uint32_t c = *(const uint16_t*)(kc + blk * kc_b + h * kc_h + off * D + d0);
        s = k_scale[blk * sc_b + h];
        x0 = code_value<FP8>(c, 0) * s;
        x1 = code_value<FP8>(c, 1) * s;
      }
    }
    TO pair[2];
    st<TO>(&pair[0], x0);
    st<TO>(&pair[1], x1);
    TO* dst = out + t * os_t + h * os_h + d0;
    if constexpr (sizeof(TO) == 2) *(uint32_t*)dst = __builtin_bit_cast(uint32_t, pair);
    else *(u32x2_t*)dst = __builtin_bit_cast(u32x2_t, pair);
  }
}

}  // namespace fdms

using namespace fdms;

// What every entry point asks of a cache: a block size 16 .. 256 that is a
// power of two, head_dim 64 or 128, 16-byte aligned blocks, slots in 31 bits.
static bool block_cache_ok(const void* kc, int64_t kc_b, int64_t kc_h, const void* vc, int64_t vc_b, int64_t vc_h,
                           int num_blocks, int block_size, int head_dim) {
  return block_size >= 16 && block_size <= 256 && (block_size & (block_size - 1)) == 0 &&
         (head_dim == 64 || head_dim == 128) && num_blocks > 0 &&
         (int64_t)num_blocks * block_size <= 0x7FFFFFFF && fdms_aligned16(kc, vc) && kc_b % 16 == 0 &&
         kc_h % 16 == 0 && vc_b % 16 == 0 && vc_h % 16 == 0;
}

FDMS_EXPORT int fdms_block_tables(const int32_t* cached_lens, const int32_t* new_lens, int num_seqs,
                                  int32_t* block_tables, int64_t bt_b, int width, const int32_t* free_blocks,
                                  int num_free_blocks, const int32_t* free_count, int block_size, int num_tokens,
                                  int32_t* slot_mapping, int64_t* positions, int32_t* cu_seqlens,
                                  int32_t* context_lens, int32_t* free_count_out, int32_t* status, void* stream) {
  if (num_seqs < 1 || num_seqs > kTabSeqs || width < 0 || num_free_blocks < 0 || num_tokens < 0 ||
      block_size < 16 || block_size > 256 || (block_size & (block_size - 1)) || free_count_out == free_count)
    return (int)hipErrorInvalidValue;
  const int groups = num_tokens ? (num_tokens - 1) / kTabTokens + 1 : 1;
  block_tables_kernel<<<groups, kTabThreads, 0, (hipStream_t)stream>>>(
      cached_lens, new_lens, num_seqs, block_tables, bt_b, width, free_blocks, num_free_blocks, free_count,
      __builtin_ctz(block_size), num_tokens, slot_mapping, positions, cu_seqlens, context_lens, free_count_out,
      status);
  FDMS_LAUNCH_CHECK();
  return 0;
}

template <typename T, int D, bool FP8>
static int launch_store(int block_size, dim3 grid, hipStream_t st, const void* k, int64_t ks_t, int64_t ks_h,
                        const void* v, int64_t vs_t, int64_t vs_h, void* kc, int64_t kc_b, int64_t kc_h, void* vc,
                        int64_t vc_b, int64_t vc_h, float* k_scale, float* v_scale, int64_t sc_b,
                        const int32_t* slots, int num_tokens, int num_blocks, int per_group) {
#define FDMS_STORE(W)                                                                                             \
  store_block_kernel<T, D, FP8, W><<<grid, 64 * W, 0, st>>>((const T*)k, ks_t, ks_h, (const T*)v, vs_t, vs_h,     \
                                                            (uint8_t*)kc, kc_b, kc_h, (uint8_t*)vc, vc_b, vc_h,   \
                                                            k_scale, v_scale, sc_b, slots, num_tokens, num_blocks, \
                                                            per_group)
  switch (block_size / kTile) {
    case 1: FDMS_STORE(1); break;
    case 2: FDMS_STORE(2); break;
    case 4: FDMS_STORE(4); break;
    case 8: FDMS_STORE(8); break;
    default: FDMS_STORE(16); break;
  }
#undef FDMS_STORE
  FDMS_LAUNCH_CHECK();
  return 0;
}

FDMS_EXPORT int fdms_store_block_kvcache(const void* key, const void* value, int dtype, int64_t ks_t, int64_t ks_h,
                                         int64_t vs_t, int64_t vs_h, void* k_cache, void* v_cache, int is_fp8,
                                         int64_t kc_b, int64_t kc_h, int64_t vc_b, int64_t vc_h, float* k_scale,
                                         float* v_scale, int64_t sc_b, const int32_t* slot_mapping, int num_tokens,
                                         int num_blocks, int block_size, int num_kv_heads, int head_dim,
                                         void* stream) {
  if (dtype < kF32 || dtype > kBF16 || num_tokens < 0 || num_kv_heads < 1 || num_kv_heads > 65535)
    return (int)hipErrorInvalidValue;
  if (!block_cache_ok(k_cache, kc_b, kc_h, v_cache, vc_b, vc_h, num_blocks, block_size, head_dim))
    return (int)hipErrorInvalidValue;
  const int64_t size = dtype == kF32 ? 4 : 2;
  if (!fdms_aligned16(key, value) || ks_t * size % 16 || ks_h * size % 16 || vs_t * size % 16 || vs_h * size % 16)
    return (int)hipErrorInvalidValue;
  if (num_tokens == 0) return 0;
  // A workgroup looks for runs in as many tokens as a block holds: a prompt's
  // workgroups then find one or two each.  A step of few tokens, whose rows
  // lie in a block each, gets a workgroup per token, so none stores several.
  const int per_group = num_tokens <= 512 ? 1 : block_size;
  const dim3 grid((num_tokens - 1) / per_group + 1, num_kv_heads, 2);
#define FDMS_ARGS                                                                                                 \
  block_size, grid, (hipStream_t)stream, key, ks_t, ks_h, value, vs_t, vs_h, k_cache, kc_b, kc_h, v_cache, vc_b,  \
      vc_h, k_scale, v_scale, sc_b, slot_mapping, num_tokens, num_blocks, per_group
  FDMS_DISPATCH_FLOAT(dtype, T, {
    if (head_dim == 64) return is_fp8 ? launch_store<T, 64, true>(FDMS_ARGS) : launch_store<T, 64, false>(FDMS_ARGS);
    return is_fp8 ? launch_store<T, 128, true>(FDMS_ARGS) : launch_store<T, 128, false>(FDMS_ARGS);
  });
#undef FDMS_ARGS
  return 0;
}

FDMS_EXPORT int fdms_gather_block_kvcache(const void* k_cache, const void* v_cache, int is_fp8, int64_t kc_b,
                                          int64_t kc_h, int64_t vc_b, int64_t vc_h, const float* k_scale,
                                          const float* v_scale, int64_t sc_b, const int32_t* slot_mapping,
                                          int num_tokens, int num_blocks, int block_size, int num_kv_heads,
                                          int head_dim, void* out_k, void* out_v, int out_dtype, int64_t ok_t,
                                          int64_t ok_h, int64_t ov_t, int64_t ov_h, void* stream) {
  if (out_dtype < kF32 || out_dtype > kBF16 || num_tokens < 0 || num_kv_heads < 1 || num_kv_heads > 65535)
    return (int)hipErrorInvalidValue;
  if (!block_cache_ok(k_cache, kc_b, kc_h, v_cache, vc_b, vc_h, num_blocks, block_size, head_dim))
    return (int)hipErrorInvalidValue;
  const int64_t pair = out_dtype == kF32 ? 8 : 4;  // bytes a lane stores
  if ((uintptr_t)out_k % pair || (uintptr_t)out_v % pair || (ok_t | ok_h | ov_t | ov_h) % 2)
    return (int)hipErrorInvalidValue;
  if (num_tokens == 0) return 0;
  const dim3 grid((num_tokens - 1) / (4 * kTile) + 1, num_kv_heads, 2);
  const int shift = __builtin_ctz(block_size);
  hipStream_t st = (hipStream_t)stream;
#define FDMS_GATHER(TT, D, F)                                                                                     \
  gather_block_kernel<TT, D, F><<<grid, 256, 0, st>>>((const uint8_t*)k_cache, kc_b, kc_h, (const uint8_t*)v_cache, \
                                                     vc_b, vc_h, k_scale, v_scale, sc_b, slot_mapping, num_tokens, \
                                                     num_blocks, shift, (TT*)out_k, ok_t, ok_h, (TT*)out_v, ov_t,  \
                                                     ov_h)
  FDMS_DISPATCH_FLOAT(out_dtype, T, {
    if (head_dim == 64) {
      if (is_fp8) FDMS_GATHER(T, 64, true);
      else FDMS_GATHER(T, 64, false);
    } else {
      if (is_fp8) FDMS_GATHER(T, 128, true);
      else FDMS_GATHER(T, 128, false);
    }
  });
#undef FDMS_GATHER
  FDMS_LAUNCH_CHECK();
  return 0;
}
