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
// in LDS.  A second launch for the map would cost more than the repeated sums:
// a kernel node of a graph takes 2.4 us here, and this one, a chain of loads
// (count and lengths, then a table or stack entry) around two barriers, 5.4 us
// for 256 decoding sequences and 6.7 for 48 prompts of 218 000 tokens.
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
  __shared__ int s_bad[kTabThreads / kWave];
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
  const int narrow = __any(bad & kTabNarrow) ? kTabNarrow : 0, invalid = __any(bad & kTabInvalid) ? kTabInvalid : 0;
  if (lane == kWave - 1) {
    s_wave[0][wave] = tinc;
    s_wave[1][wave] = binc;
    s_bad[wave] = narrow | invalid;
  }
  __syncthreads();
  int64_t tbase = tinc - tsum, bbase = binc - bsum, ttotal = 0, btotal = 0;
  int status = 0;
  for (int w = 0; w < kTabThreads / kWave; ++w) {
    if (w < wave) {
      tbase += s_wave[0][w];
      bbase += s_wave[1][w];
    }
    ttotal += s_wave[0][w];
    btotal += s_wave[1][w];
    status |= s_bad[w];
  }
  if (ttotal > num_tokens) status |= kTabTokensShort;
  if (btotal > held_free) status |= kTabNoBlocks;
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
  __syncthreads();

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
// Rows t .. t + n - 1 with consecutive slots of one block are a run, and it is
// stored, for one kv head and K or V, by the workgroup whose tokens hold its
// first row: a run inside one 16-row tile by a wave, so that a decode step's rows,
// a block each, go side by side; a longer one by the four waves, a tile at a
// time.  The rows' amax gives the block's scale before they are encoded; a wave
// keeps its last tile's rows in registers between the two and reads the others
// again, from the caches.  When the run raises the block's scale, the rows before
// it are encoded again.
//
// Bound by HBM: 4 bytes read per K and V value pair and 2 written.  What counted
// for prompts: every row's load issued before the first is looked at (a row at a
// time behind its own bounds test took 131 us where all at once take 90: 26 000
// rows of 8 heads of 128 in blocks of 256), the heads, and K and V, of the same
// tokens in neighbouring workgroups, which read whole rows of the projection (72
// -> 58: one head's rows alone lie 12 KB apart, on few memory channels), and codes
// without clamps for waves of finite values.  And for decode steps, whose runs
// have one row: a wave per run instead of a workgroup the size of a block, with
// 600 rows in blocks of 256 16.1 us instead of 688, 33 rows 4.8 instead of 11.7.
// N row elements as loaded (two to a register where they are halves), and as fp32.
template <typename T, int N>
struct Raw {
  static constexpr int W = N * (int)sizeof(T) / 4;
  uint32_t w[W];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (W % 4 == 0) {
#pragma unroll
      for (int i = 0; i < W; i += 4) {
        const u32x4_t r = *(const u32x4_t*)(p + i * 4 / sizeof(T));
#pragma unroll
        for (int j = 0; j < 4; ++j) w[i + j] = r[j];
      }
    } else if constexpr (W == 2) {
      const u32x2_t r = *(const u32x2_t*)p;
      w[0] = r[0];
      w[1] = r[1];
    } else {
      w[0] = *(const uint32_t*)p;
    }
  }
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    const uint16_t e = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
    return ld<T>((const T*)&e);
  }
};

// Codes of four values x, times inv = 1 / scale.  A wave all of whose values are
// finite needs neither clamp nor NaN test: |x| / scale is at most the largest
// code.  int8 then takes one fma per value, whose sum with 1.5 * 2^23 holds
// the rounded integer in its low byte (x / scale is exact, so it rounds once).
template <bool FP8>
__device__ __forceinline__ uint32_t encode4_finite(float a, float b, float c, float d, float inv) {
  if constexpr (FP8) {
    const uint32_t r = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, (int)r, true);
  }
  const float k = 12582912.0f;
  const uint32_t x = __float_as_uint(__builtin_fmaf(a, inv, k)), y = __float_as_uint(__builtin_fmaf(b, inv, k));
  const uint32_t z = __float_as_uint(__builtin_fmaf(c, inv, k)), w = __float_as_uint(__builtin_fmaf(d, inv, k));
  // perm selects from (second operand bytes 0-3, first operand bytes 4-7)
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(w, z, 0x0C0C0400u), __builtin_amdgcn_perm(y, x, 0x0C0C0400u),
                               0x05040100u);
}
// Four codes of a block whose scale has grown (ratio: old / new, below 1).
template <bool FP8>
__device__ __forceinline__ uint32_t encode4_again(uint32_t c, float ratio) {
  return encode4<FP8>(code_value<FP8>(c, 0) * ratio, code_value<FP8>(c, 1) * ratio, code_value<FP8>(c, 2) * ratio,
                      code_value<FP8>(c, 3) * ratio);
}

// The scale of a block after a run's rows (amax) joined `off` earlier ones.
template <bool FP8>
__device__ __forceinline__ float joined_scale(float amax, int off, float old) {
  const float need = block_scale<FP8>(amax);
  return off > 0 ? fmaxf(old, need) : need;
}

// What a run does to its block: rows off .. off + n - 1 are new.
struct Run {
  int off, n;
  float inv, ratio;  // 1 / scale; the former scale over it
  bool grown;        // the rows before are encoded again
};

// A 16-row tile of K in a wave's registers, 8 channels of some rows per lane.
template <typename T, int D, bool FP8>
struct TileK {
  static constexpr int LPR = D / 8, RPP = kWave / LPR, PASS = kTile / RPP;
  Raw<T, 8> v[PASS];
  __device__ __forceinline__ static int row() { return lane_id() / LPR; }
  __device__ __forceinline__ static int channel() { return (lane_id() % LPR) * 8; }
  __device__ __forceinline__ void load(const T* x, int64_t xs_t, int tile, int off, int n) {
    const int r0 = tile * kTile - off;
    if (r0 >= 0 && r0 + kTile <= n) {  // all rows new: one address per lane, the passes at scalar steps
      const T* p = x + (int64_t)(r0 + row()) * xs_t + channel();
#pragma unroll
      for (int i = 0; i < PASS; ++i) v[i].load(p + i * RPP * xs_t);
    } else {  // in place of rows outside the run its first or last again
#pragma unroll
      for (int i = 0; i < PASS; ++i)
        v[i].load(x + (int64_t)min(max(r0 + row() + i * RPP, 0), n - 1) * xs_t + channel());
    }
  }
  // largest magnitude; odd: NaN once a value is infinite or NaN
  __device__ __forceinline__ void look(float* amax, float* odd) const {
#pragma unroll
    for (int i = 0; i < PASS; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        *amax = fmaxf(*amax, fabsf(v[i][j]));
        *odd = __builtin_fmaf(v[i][j], 0.0f, *odd);
      }
  }
  __device__ __forceinline__ void store(uint8_t* block, int tile, const Run& run, bool finite) const {
    u32x2_t c[PASS];
    if (finite) {
#pragma unroll
      for (int i = 0; i < PASS; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          c[i][j] = encode4_finite<FP8>(v[i][4 * j], v[i][4 * j + 1], v[i][4 * j + 2], v[i][4 * j + 3], run.inv);
    } else {
#pragma unroll
      for (int i = 0; i < PASS; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          c[i][j] = encode4<FP8>(nan_to_zero(v[i][4 * j]) * run.inv, nan_to_zero(v[i][4 * j + 1]) * run.inv,
                                 nan_to_zero(v[i][4 * j + 2]) * run.inv, nan_to_zero(v[i][4 * j + 3]) * run.inv);
    }
#pragma unroll
    for (int i = 0; i < PASS; ++i) {
      const int r = tile * kTile + row() + i * RPP;
      if (r >= run.off && r < run.off + run.n) *(u32x2_t*)(block + r * D + channel()) = c[i];
    }
    if (run.grown && tile * kTile < run.off) again(block, tile, run);
  }
  // the tile's rows before the run
  __device__ __forceinline__ static void again(uint8_t* block, int tile, const Run& run) {
#pragma unroll
    for (int i = 0; i < PASS; ++i) {
      const int r = tile * kTile + row() + i * RPP;
      u32x2_t* p = (u32x2_t*)(block + r * D + channel());
      if (r < run.off) {
        u32x2_t was = *p;
        was[0] = encode4_again<FP8>(was[0], run.ratio);
        was[1] = encode4_again<FP8>(was[1], run.ratio);
        *p = was;
      }
    }
  }
};

// And of V: two channels of 16 (D = 128) or 8 (D = 64) tokens per lane, the bytes it stores.
template <typename T, int D, bool FP8>
struct TileV {
  static constexpr int LPR = D / 2, TOK = kTile * LPR / kWave, WORDS = TOK / 4;
  typedef uint32_t words_t __attribute__((ext_vector_type(WORDS)));
  static constexpr int STEP = kTile / (4 * WORDS);  // words_t's from a channel's tokens to the next one's
  Raw<T, 2> v[TOK];
  __device__ __forceinline__ static int row() { return lane_id() / LPR * TOK; }
  __device__ __forceinline__ static int channel() { return (lane_id() % LPR) * 2; }
  __device__ __forceinline__ static words_t* place(uint8_t* block, int tile) {
    return (words_t*)(block + tile * (kTile * D) + channel() * kTile + row());
  }
  __device__ __forceinline__ void load(const T* x, int64_t xs_t, int tile, int off, int n) {
    const int r0 = tile * kTile - off;
    if (r0 >= 0 && r0 + kTile <= n) {
      const T* p = x + (int64_t)(r0 + row()) * xs_t + channel();
#pragma unroll
      for (int j = 0; j < TOK; ++j) v[j].load(p + j * xs_t);
    } else {
#pragma unroll
      for (int j = 0; j < TOK; ++j) v[j].load(x + (int64_t)min(max(r0 + row() + j, 0), n - 1) * xs_t + channel());
    }
  }
  __device__ __forceinline__ void look(float* amax, float* odd) const {
#pragma unroll
    for (int j = 0; j < TOK; ++j) {
      *amax = fmaxf(*amax, fmaxf(fabsf(v[j][0]), fabsf(v[j][1])));
      *odd = __builtin_fmaf(v[j][0], 0.0f, *odd);
      *odd = __builtin_fmaf(v[j][1], 0.0f, *odd);
    }
  }
  __device__ __forceinline__ void store(uint8_t* block, int tile, const Run& run, bool finite) const {
    words_t code[2];
    if (finite) {
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int w = 0; w < WORDS; ++w)
          code[c][w] = encode4_finite<FP8>(v[4 * w][c], v[4 * w + 1][c], v[4 * w + 2][c], v[4 * w + 3][c], run.inv);
    } else {
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int w = 0; w < WORDS; ++w)
          code[c][w] = encode4<FP8>(nan_to_zero(v[4 * w][c]) * run.inv, nan_to_zero(v[4 * w + 1][c]) * run.inv,
                                    nan_to_zero(v[4 * w + 2][c]) * run.inv, nan_to_zero(v[4 * w + 3][c]) * run.inv);
    }
    words_t* p = place(block, tile);
    const int r0 = tile * kTile + row();
    if (!(r0 >= run.off && r0 + TOK <= run.off + run.n)) {
      // bytes of the rows before (encoded again if the scale grew) and of those behind
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const words_t was = p[c * STEP];
#pragma unroll
        for (int w = 0; w < WORDS; ++w) {
          const uint32_t old = run.grown ? encode4_again<FP8>(was[w], run.ratio) : was[w];
          uint32_t mixed = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = r0 + 4 * w + j;
            const uint32_t from = r < run.off ? old : (r < run.off + run.n ? code[c][w] : was[w]);
            mixed |= from & (0xFFu << (8 * j));
          }
          code[c][w] = mixed;
        }
      }
    }
    p[0] = code[0];
    p[STEP] = code[1];
  }
  __device__ __forceinline__ static void again(uint8_t* block, int tile, const Run& run) {  // all rows before the run
    words_t* p = place(block, tile);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      words_t was = p[c * STEP];
#pragma unroll
      for (int w = 0; w < WORDS; ++w) was[w] = encode4_again<FP8>(was[w], run.ratio);
      p[c * STEP] = was;
    }
  }
};

constexpr int kStoreWaves = 4;

// A run by one wave (its rows lie in one tile) or by the workgroup.
template <typename TILE, bool TEAM, bool FP8, typename T>
__device__ __forceinline__ void store_run(const T* x, int64_t xs_t, uint8_t* block, float* scale, int off, int n,
                                          float* s_red) {
  const int first = off / kTile, last = (off + n - 1) / kTile, step = TEAM ? kStoreWaves : 1;
  const int wave = TEAM ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const float old = *scale;
  TILE tile;
  float amax = 0.0f, odd = 0.0f;
  int held = -1;  // the tile in registers
  for (int i = first + wave; i <= last; i += step) {
    tile.load(x, xs_t, i, off, n);
    tile.look(&amax, &odd);
    held = i;
  }
  amax = wave_max(amax);
  if constexpr (TEAM) {
    __syncthreads();  // the last run's maxima have been read
    if (lane_id() == 0) s_red[wave] = amax;
    __syncthreads();
    amax = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
  }
  const float s = joined_scale<FP8>(amax, off, old);
  Run run;
  run.off = off, run.n = n, run.inv = 1.0f / s, run.ratio = old * run.inv, run.grown = off > 0 && s > old;
  const bool finite = !__any(odd != odd);
  for (int i = held; i >= first; i -= step) {
    if (i != held) tile.load(x, xs_t, i, off, n);
    tile.store(block, i, run, finite);
  }
  if (run.grown)
    for (int i = wave; i < first; i += step) TILE::again(block, i, run);
  if (TEAM ? threadIdx.x == 0 : lane_id() == 0) *scale = s;
}

template <typename T, int D, bool FP8>
__global__ __launch_bounds__(64 * kStoreWaves) void store_block_kernel(
    const T* __restrict__ k, int64_t ks_t, int64_t ks_h, const T* __restrict__ v, int64_t vs_t, int64_t vs_h,
    uint8_t* kc, int64_t kc_b, int64_t kc_h, uint8_t* vc, int64_t vc_b, int64_t vc_h, float* k_scale,
    float* v_scale, int64_t sc_b, const int32_t* __restrict__ slots, int num_tokens, int num_blocks, int shift,
    int num_heads, int tokens) {
  __shared__ float s_red[kStoreWaves];
  __shared__ int s_long[kStoreWaves * kWave][3];  // runs for the workgroup: first token, its slot, rows
  __shared__ int s_count;
  // heads, and K and V, run fastest: workgroups that run together read whole rows of the projection
  const unsigned heads2 = 2 * num_heads, part = blockIdx.x % heads2;
  const int h = part % num_heads, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool is_v = part >= (unsigned)num_heads;
  const T* x = is_v ? v + h * vs_h : k + h * ks_h;
  const int64_t xs_t = is_v ? vs_t : ks_t, c_b = is_v ? vc_b : kc_b;
  uint8_t* base = is_v ? vc + h * vc_h : kc + h * kc_h;
  float* scale = (is_v ? v_scale : k_scale) + h;
  const int bs = 1 << shift;
  // lane i looks at the wave's token i: does a run begin there?
  const int64_t t0 = ((int64_t)(blockIdx.x / heads2) * kStoreWaves + wave) * tokens, mine = t0 + lane;
  const bool here = lane < tokens && mine < num_tokens;
  const int slot_l = here ? slots[mine] : -1, before = here && mine > 0 ? slots[mine - 1] : -1;
  const bool leads = slot_l >= 0 && (slot_l >> shift) < num_blocks &&
                     ((slot_l & (bs - 1)) == 0 || mine == 0 || before != slot_l - 1);
  uint64_t leaders = __ballot(leads);
  if (threadIdx.x == 0) s_count = 0;
  __syncthreads();
  while (leaders) {
    const int i = __builtin_ctzll(leaders);
    leaders &= leaders - 1;
    const int slot = __builtin_amdgcn_readlane(slot_l, i), off = slot & (bs - 1);
    const int64_t t = t0 + i;
    int n = 0;  // the leading rows whose slots follow on, all looked up at once
    constexpr int LOOKS = (1 << kMaxBlockLog2) / kWave;
    int seen[LOOKS];
#pragma unroll
    for (int j = 0; j < LOOKS; ++j)
      seen[j] = j == 0 || j * kWave < bs ? slots[min(t + j * kWave + lane, (int64_t)num_tokens - 1)] : -1;
    bool whole = true;
#pragma unroll
    for (int j = 0; j < LOOKS; ++j) {
      const int at = j * kWave + lane;
      const uint64_t m = ~__ballot(off + at < bs && t + at < num_tokens && seen[j] == slot + at);
      const int rows = m ? __builtin_ctzll(m) : kWave;
      n += whole ? rows : 0;
      whole = whole && rows == kWave;
    }
    if (off / kTile == (off + n - 1) / kTile) {
      const int64_t blk = slot >> shift;
      if (is_v)
        store_run<TileV<T, D, FP8>, false, FP8>(x + t * xs_t, xs_t, base + blk * c_b, scale + blk * sc_b, off, n, s_red);
      else
        store_run<TileK<T, D, FP8>, false, FP8>(x + t * xs_t, xs_t, base + blk * c_b, scale + blk * sc_b, off, n, s_red);
    } else if (lane == 0) {
      const int at = atomicAdd(&s_count, 1);  // (whatever their order, the runs are independent)
      s_long[at][0] = (int)t;
      s_long[at][1] = slot;
      s_long[at][2] = n;
    }
  }
  __syncthreads();
  for (int j = 0; j < s_count; ++j) {
    const int64_t t = __builtin_amdgcn_readfirstlane(s_long[j][0]);
    const int slot = __builtin_amdgcn_readfirstlane(s_long[j][1]), n = __builtin_amdgcn_readfirstlane(s_long[j][2]);
    const int64_t blk = slot >> shift;
    const int off = slot & (bs - 1);
    if (is_v)
      store_run<TileV<T, D, FP8>, true, FP8>(x + t * xs_t, xs_t, base + blk * c_b, scale + blk * sc_b, off, n, s_red);
    else
      store_run<TileK<T, D, FP8>, true, FP8>(x + t * xs_t, xs_t, base + blk * c_b, scale + blk * sc_b, off, n, s_red);
  }
}

// ------------------------------------------------------------------ read-back
// Dense rows of the tokens at slots[t]; a slot outside the cache gives zeros.
// A wave takes 16 tokens of one kv head, K or V, every load on its way before
// the first is looked at.  K: 16 bytes of a row per lane.  V comes from
// transposed tiles: a lane holds the 16 tokens of two channels of the tiles that
// its first and last token lie in -- a run of slots has no others -- and looks up
// single bytes of any further ones.  27 000 rows of 8 x 128 39 us (4.3 TB/s),
// 17 000 of 8 x 64 16 us (3.4); a token at a time 54 and 25.
// Two values as TO's, to nearest even by the hardware (v_cvt_pk_bf16_f32, v_cvt_pk_f16_f32).
template <typename TO> struct Pair;
template <> struct Pair<float> {
  typedef u32x2_t bits;
  static __device__ __forceinline__ bits of(float a, float b) { return bits{__float_as_uint(a), __float_as_uint(b)}; }
};
template <> struct Pair<f16_t> {
  typedef uint32_t bits;
  static __device__ __forceinline__ bits of(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{a, b}), f16x2_t));
  }
};
template <> struct Pair<bf16_t> {
  typedef uint32_t bits;
  typedef __bf16 two __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ bits of(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{a, b}), two));
  }
};

// The 8-bit codes' values exactly, by the hardware's conversion (e4m3fn) or a byte's (int8).
template <bool FP8, int I>
__device__ __forceinline__ float code_value_at(uint32_t c) {
  if constexpr (FP8) return __builtin_amdgcn_cvt_f32_fp8((int)c, I);
  return (float)((int)(c << (24 - 8 * I)) >> 24);
}

template <typename TO, int D, bool FP8>
__global__ __launch_bounds__(256) void gather_block_kernel(
    const uint8_t* __restrict__ kc, int64_t kc_b, int64_t kc_h, const uint8_t* __restrict__ vc, int64_t vc_b,
    int64_t vc_h, const float* __restrict__ k_scale, const float* __restrict__ v_scale, int64_t sc_b,
    const int32_t* __restrict__ slots, int num_tokens, int num_blocks, int shift, TO* __restrict__ out_k,
    int64_t ok_t, int64_t ok_h, TO* __restrict__ out_v, int64_t ov_t, int64_t ov_h, int num_heads) {
  const unsigned chunks = gridDim.x / (2u * num_heads), part = blockIdx.x / chunks;
  const int h = part % num_heads, lane = lane_id(), mask = (1 << shift) - 1;
  const bool is_v = part >= (unsigned)num_heads;
  const int64_t first = ((int64_t)(blockIdx.x % chunks) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * kTile;
  if (first >= num_tokens) return;
  const int left = (int)min((int64_t)num_tokens - first, (int64_t)kTile);
  // lane i holds token i % 16: its slot (-1 outside the cache) and scale
  int slot = slots[first + min(lane & 15, left - 1)];
  if (slot < 0 || slot >> shift >= num_blocks) slot = -1;
  const float* scales = is_v ? v_scale : k_scale;
  const float sc = slot < 0 ? 0.0f : scales[(int64_t)(slot >> shift) * sc_b + h];
  if (!is_v) {
    constexpr int LPR = D / 16, RPP = kWave / LPR, PASS = kTile / RPP;
    u32x4_t c[PASS];
    int sl[PASS];
    float s[PASS];
#pragma unroll
    for (int i = 0; i < PASS; ++i) {
      const int row = i * RPP + lane / LPR;
      sl[i] = __shfl(slot, row, kWave);
      s[i] = __shfl(sc, row, kWave);
      const int at = max(sl[i], 0);
      c[i] = *(const u32x4_t*)(kc + (int64_t)(at >> shift) * kc_b + h * kc_h + (at & mask) * D + (lane % LPR) * 16);
    }
#pragma unroll
    for (int i = 0; i < PASS; ++i) {
      const int row = i * RPP + lane / LPR;
      if (row >= left) continue;
      TO* dst = out_k + (first + row) * ok_t + h * ok_h + (lane % LPR) * 16;
      typename Pair<TO>::bits e[8];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t x = sl[i] < 0 ? 0u : c[i][w];
        e[2 * w] = Pair<TO>::of(code_value_at<FP8, 0>(x) * s[i], code_value_at<FP8, 1>(x) * s[i]);
        e[2 * w + 1] = Pair<TO>::of(code_value_at<FP8, 2>(x) * s[i], code_value_at<FP8, 3>(x) * s[i]);
      }
#pragma unroll
      for (int w = 0; w < (int)sizeof(TO); ++w) ((u32x4_t*)dst)[w] = ((const u32x4_t*)e)[w];
    }
    return;
  }
  constexpr int LPR = D / 2, TOK = kTile * LPR / kWave;  // lanes per row, tokens per lane
  const int t0 = (lane / LPR) * TOK, d0 = (lane % LPR) * 2;
  auto tile_at = [&](int s) {  // the lane's channels of the tile that holds a slot
    const int at = max(s, 0);
    return (const u32x4_t*)(vc + (int64_t)(at >> shift) * vc_b + h * vc_h + ((at & mask) >> 4) * (D * kTile) +
                            d0 * kTile);
  };
  int sl[TOK];
  float s[TOK];
#pragma unroll
  for (int j = 0; j < TOK; ++j) {
    sl[j] = __shfl(slot, t0 + j, kWave);
    s[j] = __shfl(sc, t0 + j, kWave);
  }
  const int a_tile = sl[0] >> 4, b_tile = sl[TOK - 1] >> 4;
  const u32x4_t a0 = tile_at(sl[0])[0], a1 = tile_at(sl[0])[1];
  const u32x4_t b0 = tile_at(sl[TOK - 1])[0], b1 = tile_at(sl[TOK - 1])[1];
#pragma unroll
  for (int j = 0; j < TOK; ++j) {
    if (t0 + j >= left) break;
    const int tile = sl[j] >> 4, w = (sl[j] >> 2) & 3, sh = 8 * (sl[j] & 3);
    uint32_t x, y;
    if (tile == a_tile || tile == b_tile) {
      const u32x4_t c0 = tile == a_tile ? a0 : b0, c1 = tile == a_tile ? a1 : b1;
      x = (w & 2 ? (w & 1 ? c0[3] : c0[2]) : (w & 1 ? c0[1] : c0[0])) >> sh;
      y = (w & 2 ? (w & 1 ? c1[3] : c1[2]) : (w & 1 ? c1[1] : c1[0])) >> sh;
    } else {
      const uint8_t* p = (const uint8_t*)tile_at(sl[j]) + (sl[j] & 15);
      x = p[0];
      y = p[kTile];
    }
    if (sl[j] < 0) x = y = 0;
    *(typename Pair<TO>::bits*)(out_v + (first + t0 + j) * ov_t + h * ov_h + d0) =
        Pair<TO>::of(code_value_at<FP8, 0>(x) * s[j], code_value_at<FP8, 0>(y) * s[j]);
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

// Whether [a, a + n) and [b, b + m) of elements of the given sizes meet.
inline bool meet(const void* a, int64_t n, int size_a, const void* b, int64_t m, int size_b) {
  const char *p = (const char*)a, *q = (const char*)b;
  return n > 0 && m > 0 && p < q + m * size_b && q < p + n * size_a;
}

FDMS_EXPORT int fdms_block_tables(const int32_t* cached_lens, const int32_t* new_lens, int num_seqs,
                                  int32_t* block_tables, int64_t bt_b, int width, const int32_t* free_blocks,
                                  int num_free_blocks, const int32_t* free_count, int block_size, int num_tokens,
                                  int32_t* slot_mapping, int64_t* positions, int32_t* cu_seqlens,
                                  int32_t* context_lens, int32_t* free_count_out, int32_t* status, void* stream) {
  if (num_seqs < 1 || num_seqs > kTabSeqs || width < 0 || num_free_blocks < 0 || num_tokens < 0 ||
      block_size < 16 || block_size > 256 || (block_size & (block_size - 1)))
    return (int)hipErrorInvalidValue;
  // workgroups read the inputs while others write the outputs
  const struct {
    const void* at;
    int64_t n;
    int size;
  } in[] = {{cached_lens, num_seqs, 4}, {new_lens, num_seqs, 4}, {block_tables, (num_seqs - 1) * bt_b + width, 4},
            {free_blocks, num_free_blocks, 4}, {free_count, 1, 4}},
    out[] = {{slot_mapping, num_tokens, 4}, {positions, num_tokens, 8}, {cu_seqlens, num_seqs + 1, 4},
             {context_lens, num_seqs, 4}, {free_count_out, 1, 4}, {status, 1, 4}};
  for (const auto& i : in)
    for (const auto& o : out)
      if (meet(i.at, i.n, i.size, o.at, o.n, o.size)) return (int)hipErrorInvalidValue;
  const int groups = num_tokens ? (num_tokens - 1) / kTabTokens + 1 : 1;
  block_tables_kernel<<<groups, kTabThreads, 0, (hipStream_t)stream>>>(
      cached_lens, new_lens, num_seqs, block_tables, bt_b, width, free_blocks, num_free_blocks, free_count,
      __builtin_ctz(block_size), num_tokens, slot_mapping, positions, cu_seqlens, context_lens, free_count_out,
      status);
  FDMS_LAUNCH_CHECK();
  return 0;
}

FDMS_EXPORT int fdms_store_block_kvcache(const void* key, const void* value, int dtype, int64_t ks_t, int64_t ks_h,
                                         int64_t vs_t, int64_t vs_h, void* k_cache, void* v_cache, int is_fp8,
                                         int64_t kc_b, int64_t kc_h, int64_t vc_b, int64_t vc_h, float* k_scale,
                                         float* v_scale, int64_t sc_b, const int32_t* slot_mapping, int num_tokens,
                                         int num_blocks, int block_size, int num_kv_heads, int head_dim,
                                         void* stream) {
  if (dtype < kF32 || dtype > kBF16 || num_tokens < 0 || num_kv_heads < 1 ||
      ((int64_t)num_tokens / 64 + 512) * 2 * num_kv_heads > 0x7FFFFFFF)  // workgroups of the grid
    return (int)hipErrorInvalidValue;
  if (!block_cache_ok(k_cache, kc_b, kc_h, v_cache, vc_b, vc_h, num_blocks, block_size, head_dim))
    return (int)hipErrorInvalidValue;
  const int64_t size = dtype == kF32 ? 4 : 2;
  if (!fdms_aligned16(key, value) || ks_t * size % 16 || ks_h * size % 16 || vs_t * size % 16 || vs_h * size % 16)
    return (int)hipErrorInvalidValue;
  if (num_tokens == 0) return 0;
  // Tokens whose runs a wave looks for, at most one for each of its lanes: one
  // where they may be a decode step's, with a run each, then so many that the
  // grid has the 4096 waves the card holds (8 heads of 128, blocks of 256: 2000
  // decode rows 45 us and a run of 2000 rows 8.8; with twice the waves 42 and 11.7,
  // with half 62 and 9.1; with a token a wave 44 and 15), up to a block's or 64 per
  // workgroup, past which workgroups would have several long runs to store.
  const int most = block_size <= 64 ? 16 : block_size / 4;
  const int tokens = (int)std::min<int64_t>(std::max<int64_t>((int64_t)num_tokens * 2 * num_kv_heads / 4096, 1), most);
  const dim3 grid(((num_tokens - 1) / (tokens * kStoreWaves) + 1) * 2u * num_kv_heads);
#define FDMS_STORE(TT, D, F)                                                                                       \
  store_block_kernel<TT, D, F><<<grid, 64 * kStoreWaves, 0, (hipStream_t)stream>>>(                                \
      (const TT*)key, ks_t, ks_h, (const TT*)value, vs_t, vs_h, (uint8_t*)k_cache, kc_b, kc_h, (uint8_t*)v_cache,  \
      vc_b, vc_h, k_scale, v_scale, sc_b, slot_mapping, num_tokens, num_blocks, __builtin_ctz(block_size),         \
      num_kv_heads, tokens)
  FDMS_DISPATCH_FLOAT(dtype, T, {
    if (head_dim == 64) {
      if (is_fp8) FDMS_STORE(T, 64, true);
      else FDMS_STORE(T, 64, false);
    } else {
      if (is_fp8) FDMS_STORE(T, 128, true);
      else FDMS_STORE(T, 128, false);
    }
  });
#undef FDMS_STORE
  FDMS_LAUNCH_CHECK();
  return 0;
}

FDMS_EXPORT int fdms_gather_block_kvcache(const void* k_cache, const void* v_cache, int is_fp8, int64_t kc_b,
                                          int64_t kc_h, int64_t vc_b, int64_t vc_h, const float* k_scale,
                                          const float* v_scale, int64_t sc_b, const int32_t* slot_mapping,
                                          int num_tokens, int num_blocks, int block_size, int num_kv_heads,
                                          int head_dim, void* out_k, void* out_v, int out_dtype, int64_t ok_t,
                                          int64_t ok_h, int64_t ov_t, int64_t ov_h, void* stream) {
  if (out_dtype < kF32 || out_dtype > kBF16 || num_tokens < 0 || num_kv_heads < 1 ||
      ((int64_t)num_tokens / 64 + 512) * 2 * num_kv_heads > 0x7FFFFFFF)  // workgroups of the grid
    return (int)hipErrorInvalidValue;
  if (!block_cache_ok(k_cache, kc_b, kc_h, v_cache, vc_b, vc_h, num_blocks, block_size, head_dim))
    return (int)hipErrorInvalidValue;
  if (!fdms_aligned16(out_k, out_v) || (ok_t | ok_h | ov_t | ov_h) % 8) return (int)hipErrorInvalidValue;
  if (num_tokens == 0) return 0;
  const dim3 grid(((num_tokens - 1) / (4 * kTile) + 1) * 2u * num_kv_heads);
  const int shift = __builtin_ctz(block_size);
  hipStream_t st = (hipStream_t)stream;
#define FDMS_GATHER(TT, D, F)                                                                                     \
  gather_block_kernel<TT, D, F><<<grid, 256, 0, st>>>((const uint8_t*)k_cache, kc_b, kc_h, (const uint8_t*)v_cache, \
                                                     vc_b, vc_h, k_scale, v_scale, sc_b, slot_mapping, num_tokens, \
                                                     num_blocks, shift, (TT*)out_k, ok_t, ok_h, (TT*)out_v, ov_t,  \
                                                     ov_h, num_kv_heads)
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
