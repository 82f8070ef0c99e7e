// A cache in 4 bits (kv4.cuh): keys and values written and read back, and tokens dropped by the weights they gathered.
#include "kv4.cuh"

#define GB_MAX_GRID_YZ 65535

struct Kv4RowsArgs {
  const void* kv;          // [T, 2 nkv, D]: what is written, or (out) what is read
  void* out;
  const int* token_seq;    // [T]
  const int* token_pos;    // [T], or null: a row is one of its sequence's newest tokens, by kv_len and cu_q
  const int* slots;        // [n_seqs]
  const int* block_table;  // [n_slots, max_pages]
  const int* kv_len;       // [n_seqs]
  const int* cu_q;         // [n_seqs + 1]
  uint8_t* pages;
  float* weights;          // [n_pages, nkv, 64] set to 0 for the tokens written, or null
  int T, n_seqs, n_slots, nkv, max_pages, n_pages;
};

// Where token t of a step lives: its page (-1: nowhere) and its place there.
__device__ __forceinline__ int find_token(const Kv4RowsArgs& a, int t, int& place) {
  const int seq = a.token_seq[t];
  place = 0;
  if ((unsigned)seq >= (unsigned)a.n_seqs) return -1;
  const int pos = a.token_pos ? a.token_pos[t] : a.kv_len[seq] - (a.cu_q[seq + 1] - t);
  if (pos < 0) return -1;
  place = pos & (KV4_PAGE - 1);
  const int slot = a.slots[seq];
  if ((unsigned)slot >= (unsigned)a.n_slots) return -1;
  return kv4_page(a.block_table + (size_t)slot * a.max_pages, pos / KV4_PAGE, a.max_pages, a.n_pages);
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]);
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&x)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
template <>
__device__ __forceinline__ void load8<bf16>(const bf16* p, float (&x)[8]) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]);
template <>
__device__ __forceinline__ void store8<float>(float* p, const float (&x)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
template <>
__device__ __forceinline__ void store8<bf16>(bf16* p, const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<uint32_t*>(&v);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// The bits of the bfloat16 number next to x on the side of larger magnitude (x itself when it is one).
__device__ __forceinline__ uint32_t bf16_away(float x) { return (__float_as_uint(x) + 0xffffu) >> 16; }

// The code of x - m = d in steps of s: the nearest whole number to d / s, of two equally near ones the even one.  The
// product with the inverse is off by a few units of its last place, so its whole number can be wrong by one where d / s
// lies that close to the middle of two; the remainder d - c s, which one multiply-add gives to its last place, says so.
// (A rounded quotient takes a long way round for d = 0, which every group has: a step's rows of 64 tokens took 11 us.)
__device__ __forceinline__ uint32_t nearest_code(float d, float s, float inv, float half) {
  const float c = rintf(d * inv);
  const float rest = fmaf(-c, s, d);
  const int k = (int)c, odd = k & 1;
  const int up = rest > half || (odd && rest == half), down = rest < -half || (odd && rest == -half);
  return (uint32_t)min(max(k + up - down, 0), 15);
}

// Eight lanes take a group of 64 elements, a word's eight each: the group's range is three exchanges, its codes and
// pair are written straight to their places.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_write_kernel(const Kv4RowsArgs a) {
  using F = Kv4<D>;
  pdl_wait();
  const unsigned group = blockIdx.x * 32 + (threadIdx.x >> 3), heads = 2 * a.nkv;
  const int lane8 = threadIdx.x & 7;
  if (group >= (unsigned)a.T * heads * F::NG) return;          // (whole groups of lanes leave; fits 32 bits)
  const uint32_t mask = 0xffu << (threadIdx.x & 24);
  const unsigned g = group % F::NG, row = group / F::NG;
  const int t = row / heads, hh = row - t * heads;
  float x[8];
  load8(reinterpret_cast<const T*>(a.kv) + (size_t)row * D + g * KV4_GROUP + lane8 * 8, x);
  int place;
  const int page = find_token(a, t, place);
  if (page < 0) return;                                         // (the same for the group's lanes)
  float lo = x[0], hi = x[0];
  bool fine = true;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    lo = fminf(lo, x[e]), hi = fmaxf(hi, x[e]);
    fine = fine && isfinite(x[e]);
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(mask, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(mask, hi, o));
  }
  fine = __ballot_sync(mask, fine) == mask;
  const uint32_t mb = lo < 0.f ? bf16_away(lo) : __float_as_uint(lo) >> 16;      // towards minus infinity
  const float m = __uint_as_float(mb << 16);
  const uint32_t sb = bf16_away(__fdiv_rn(__fsub_rn(hi, m), 15.f));               // upwards: it is not negative
  const float s = __uint_as_float(sb << 16);
  uint32_t word = 0, pair = (mb << 16) | sb;
  // (the step is rounded up: m + 15 s may be no number where the largest element still is one)
  if (!fine || !isfinite(s) || !isfinite(m) || !(fmaf(15.f, s, m) < 0x1.FFp127f)) {        // (half a step beyond bfloat16's last)
    pair = 0x7fff7fffu;                                         // NaN, NaN
  } else if (s > 0.f) {
    // (steps at the ends of the numbers' range are brought to its middle by a power of two, exactly)
    const float scale = s < 1e-30f ? 0x1p100f : s > 1e30f ? 0x1p-100f : 1.f;
    const float s1 = s * scale, inv = __fdividef(1.f, s1), half = 0.5f * s1;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      word |= nearest_code(__fsub_rn(x[e], m) * scale, s1, inv, half) << (((e & 1) << 4) + ((e >> 1) << 2));
  }
  const bool is_v = hh >= a.nkv;
  const int h = is_v ? hh - a.nkv : hh, tok = place & (KV4_TOKENS - 1), n = g * 8 + lane8;
  uint8_t* rec = a.pages + (((size_t)page * a.nkv + h) * (KV4_PAGE / KV4_TOKENS) + place / KV4_TOKENS) * F::RECORD;
  uint32_t* codes = reinterpret_cast<uint32_t*>(rec + (is_v ? F::V_OFF : 0) + tok * F::ROW);
  codes[is_v ? F::value_word(n, tok) : F::key_word(n)] = word;
  if (lane8 == 0) {
    reinterpret_cast<uint32_t*>(rec + F::PAIR_OFF + tok * F::PAIR)[(is_v ? F::NG : 0) + g] = pair;
    if (a.weights && is_v && g == 0) a.weights[((size_t)page * a.nkv + h) * KV4_PAGE + place] = 0.f;
  }
}

#define ROWS_WARPS 4
#define ROWS_AT_ONCE 4

// The other way: a word and its pair in, eight elements out (zeros for a token that is nowhere).  A warp has a token,
// finds once where it lives and has ROWS_AT_ONCE turns' loads on their way together.  (A thread for every word, which
// found the token for itself by four loads in a row, read 16,384 tokens of 8 heads of 128 in 29.3 us, this in 16.8: 86 MB
// at 5.1 TB/s.)
template <typename T, int D>
__global__ void __launch_bounds__(32 * ROWS_WARPS) kv4_read_kernel(const Kv4RowsArgs a) {
  using F = Kv4<D>;
  pdl_wait();
  const int t = blockIdx.x * ROWS_WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (t >= a.T) return;
  const int words = 2 * a.nkv * (D / 8);
  T* out = reinterpret_cast<T*>(a.out) + (size_t)t * words * 8;
  int place;
  const int page = find_token(a, t, place);
  const int tok = place & (KV4_TOKENS - 1);
  const uint8_t* first = a.pages + ((size_t)max(page, 0) * a.nkv * (KV4_PAGE / KV4_TOKENS) + place / KV4_TOKENS) * F::RECORD;
  for (int i0 = lane; i0 < words; i0 += 32 * ROWS_AT_ONCE) {
    uint32_t w[ROWS_AT_ONCE], pair[ROWS_AT_ONCE];
#pragma unroll
    for (int u = 0; u < ROWS_AT_ONCE; ++u) {
      const int i = i0 + 32 * u, hh = i / (D / 8), n = i % (D / 8);
      w[u] = pair[u] = 0u;
      if (i < words && page >= 0) {
        const bool is_v = hh >= a.nkv;
        const uint8_t* rec = first + (size_t)(is_v ? hh - a.nkv : hh) * (KV4_PAGE / KV4_TOKENS) * F::RECORD;
        const uint32_t* codes = reinterpret_cast<const uint32_t*>(rec + (is_v ? F::V_OFF : 0) + tok * F::ROW);
        w[u] = codes[is_v ? F::value_word(n, tok) : F::key_word(n)];
        pair[u] = reinterpret_cast<const uint32_t*>(rec + F::PAIR_OFF + tok * F::PAIR)[(is_v ? F::NG : 0) + n / 8];
      }
    }
#pragma unroll
    for (int u = 0; u < ROWS_AT_ONCE; ++u) {
      if (i0 + 32 * u >= words) break;
      float x[8];
      kv4_values(w[u], pair[u], x);
      store8(out + (size_t)(i0 + 32 * u) * 8, x);
    }
  }
}

template <typename T, int D>
static int launch_rows(const Kv4RowsArgs& a, bool write, cudaStream_t s) {
  if (!write)
    return gb_launch(kv4_read_kernel<T, D>, dim3((a.T + ROWS_WARPS - 1) / ROWS_WARPS), dim3(32 * ROWS_WARPS), 0, s, a);
  const long long groups = (long long)a.T * 2 * a.nkv * (D / KV4_GROUP), blocks = (groups + 31) / 32;
  if (groups > 0x7fffffffll) return GB_ERR_UNSUPPORTED;
  return gb_launch(kv4_write_kernel<T, D>, dim3((unsigned)blocks), dim3(256), 0, s, a);
}
static int rows(const Kv4RowsArgs* a, int D, int f32, bool write, cudaStream_t s) {
  if (a->T < 0 || a->nkv <= 0 || a->max_pages <= 0 || a->n_pages <= 0 || a->n_seqs < 0 || a->n_slots < 0 || !a->pages ||
      a->T > 0x7fffff00 || a->nkv > 0x100000)
    return GB_ERR_BAD_ARG;
  if (((uintptr_t)(write ? a->kv : a->out) | (uintptr_t)a->pages) & 15) return GB_ERR_BAD_ARG;
  if (a->T == 0) return 0;
  if (!a->token_seq || !a->slots || !a->block_table || (!a->token_pos && (!a->kv_len || !a->cu_q))) return GB_ERR_BAD_ARG;
  if (D == 64) return f32 ? launch_rows<float, 64>(*a, write, s) : launch_rows<bf16, 64>(*a, write, s);
  if (D == 128) return f32 ? launch_rows<float, 128>(*a, write, s) : launch_rows<bf16, 128>(*a, write, s);
  return GB_ERR_UNSUPPORTED;
}
GB_EXPORT int gb_kv4_write(const Kv4RowsArgs* a, int D, int f32, cudaStream_t s) { return rows(a, D, f32, true, s); }
GB_EXPORT int gb_kv4_read(const Kv4RowsArgs* a, int D, int f32, cudaStream_t s) { return rows(a, D, f32, false, s); }

// ---------------------------------------------------------------- eviction
struct Kv4ChooseArgs {
  const float* weights;    // [n_pages, nkv, 64]
  const int* block_table;  // [n_slots, max_pages]
  const int* slots;        // [n_seqs]
  const int* kv_len;       // [n_seqs]
  int* kept;               // [n_seqs, nkv, keep]
  int* new_len;            // [n_seqs]
  int n_seqs, n_slots, nkv, max_pages, n_pages, keep, recent, first;
};

// A number that is larger when the weight is (a NaN above infinity; zeros of both signs are equal).
__device__ __forceinline__ uint32_t ordered(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

#define CHOOSE_THREADS 1024
#define CHOOSE_WARPS (CHOOSE_THREADS / 32)
#define CHOOSE_BINS 2048
#define CHOOSE_HELD (40 * 1024)      // the most weights that a block holds in shared memory; those behind are read again

// A whole block finds the largest digit d for which at least `left` of the counted weights have a digit >= d, and how
// many are above it: the threads have a few bins each, from the largest down.
__device__ __forceinline__ void find_digit(const int* hist, int bins, int left, int* warp_sums, int* found) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, each = bins / CHOOSE_THREADS;
  int mine = 0;
  for (int i = 0; i < each; ++i) mine += hist[bins - 1 - tid * each - i];
  int sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += v;
  }
  if (lane == 31) warp_sums[warp] = sum;
  __syncthreads();
  int before = __reduce_add_sync(0xffffffffu, lane < warp ? warp_sums[lane] : 0) + sum - mine;
  if (before < left && before + mine >= left) {
    int i = 0;
    for (;; ++i) {
      const int n = hist[bins - 1 - tid * each - i];
      if (before + n >= left) break;
      before += n;
    }
    found[0] = bins - 1 - tid * each - i, found[1] = left - before;
  }
  __syncthreads();
}

// One block chooses for one kv head of one sequence.  The weights are read once and held in shared memory; the one of
// the last token that is kept among the candidates is found digit by digit (11, 11 and 10 bits, a histogram each).  Each
// warp then has a stretch of the tokens: it counts those above that weight and those equal to it, and writes the places
// of the kept ones behind those of the warps in front of it, with the first of those that are equal to the last kept.
__global__ void __launch_bounds__(CHOOSE_THREADS) kv4_choose_kernel(const Kv4ChooseArgs a, int held) {
  extern __shared__ uint32_t held_s[];
  __shared__ int hist[CHOOSE_BINS];
  __shared__ int sums[2][CHOOSE_WARPS];
  __shared__ int found[2];
  pdl_wait();
  const int h = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int slot = a.slots[seq];
  const bool live = (unsigned)slot < (unsigned)a.n_slots;
  const int len = live ? max(0, min(a.kv_len[seq], a.max_pages * KV4_PAGE)) : 0;
  const int keep = min(a.keep, len);
  int* kept = a.kept + ((size_t)seq * a.nkv + h) * a.keep;
  if (h == 0 && tid == 0) a.new_len[seq] = keep;
  for (int i = keep + tid; i < a.keep; i += CHOOSE_THREADS) kept[i] = -1;
  if (keep == len) {
    for (int i = tid; i < len; i += CHOOSE_THREADS) kept[i] = i;
    return;
  }
  const int* table = a.block_table + (size_t)slot * a.max_pages;
  const int c0 = a.first, c1 = len - a.recent;          // the candidates; first + recent <= keep < len
  const int need = keep - a.first - a.recent;
  auto read = [&](int i) -> uint32_t {
    const int page = kv4_page(table, i / KV4_PAGE, a.max_pages, a.n_pages);
    return page < 0 ? 0u : ordered(a.weights[((size_t)page * a.nkv + h) * KV4_PAGE + (i & (KV4_PAGE - 1))]);
  };
  auto weight = [&](int i) -> uint32_t { return i < held ? held_s[i] : read(i); };
  uint32_t last = 0;                                    // the weight of the last one kept, from its top digit down
  int left = need;                                      // how many of that weight are kept
#pragma unroll 1
  for (int pass = 0; pass < 3 && need > 0; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
    for (int i = tid; i < bins; i += CHOOSE_THREADS) hist[i] = 0;
    __syncthreads();
    if (pass == 0) {
      for (int i0 = c0 + tid; i0 < c1; i0 += 4 * CHOOSE_THREADS) {      // (four loads on their way at a time)
        uint32_t u[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) u[k] = i0 + k * CHOOSE_THREADS < c1 ? read(i0 + k * CHOOSE_THREADS) : 0u;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int i = i0 + k * CHOOSE_THREADS;
          if (i >= c1) break;
          if (i < held) held_s[i] = u[k];
          atomicAdd(&hist[u[k] >> 21], 1);
        }
      }
    } else {
      const int done = pass == 1 ? 21 : 10;
      for (int i = c0 + tid; i < c1; i += CHOOSE_THREADS) {
        const uint32_t u = weight(i);
        if (u >> done == last >> done) atomicAdd(&hist[(u >> shift) & (bins - 1)], 1);
      }
    }
    __syncthreads();
    find_digit(hist, bins, left, sums[0], found);
    last |= (uint32_t)found[0] << shift;
    left = found[1];
    __syncthreads();
  }
  // warp w has tokens [w each, (w + 1) each)
  const int each = (len + CHOOSE_THREADS - 1) / CHOOSE_THREADS * 32, begin = warp * each, end = min(len, begin + each);
  auto kind = [&](int i, bool& sure, bool& tie) {       // kept whatever the others are; or equal to the last one kept
    sure = i < end && (i < c0 || i >= c1);
    tie = false;
    if (i < end && !sure && need > 0) {
      const uint32_t u = weight(i);
      sure = u > last, tie = u == last;
    }
  };
  int n_sure = 0, n_tie = 0;
  for (int i = begin + lane; i - lane < end; i += 32) {
    bool sure, tie;
    kind(i, sure, tie);
    n_sure += __popc(__ballot_sync(0xffffffffu, sure)), n_tie += __popc(__ballot_sync(0xffffffffu, tie));
  }
  if (lane == 0) sums[0][warp] = n_sure, sums[1][warp] = n_tie;
  __syncthreads();
  int ties_before, out;
  {
    const int t_all = sums[1][lane], s_all = sums[0][lane];
    int t_sum = t_all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, t_sum, o);
      if (lane >= o) t_sum += v;
    }
    const int before = t_sum - t_all;                   // of warp `lane`
    const int taken = s_all + min(max(left - before, 0), t_all);
    out = __reduce_add_sync(0xffffffffu, lane < warp ? taken : 0);
    ties_before = __shfl_sync(0xffffffffu, before, warp);
  }
  for (int i = begin + lane; i - lane < end; i += 32) {
    bool sure, tie;
    kind(i, sure, tie);
    const uint32_t ties = __ballot_sync(0xffffffffu, tie);
    const bool mine = sure || (tie && ties_before + __popc(ties & ((1u << lane) - 1)) < left);
    const uint32_t who = __ballot_sync(0xffffffffu, mine);
    if (mine) kept[out + __popc(who & ((1u << lane) - 1))] = i;
    out += __popc(who);
    ties_before += __popc(ties);
  }
}

struct Kv4MoveArgs {
  const uint8_t* from;     // pages, or records [n_seqs, nkv, keep / 16 up] one after the other (from_table null)
  uint8_t* to;
  const float* w_from;     // weights [pages, nkv, 64], or [n_seqs, nkv, keep up to 16] (from_table null)
  float* w_to;
  const int* from_table;   // [n_slots, from_max]
  const int* to_table;     // [n_slots, to_max]
  const int* slots;        // [n_seqs]
  const int* kept;         // [n_seqs, nkv, keep], -1 behind the last
  int n_seqs, n_slots, nkv, n_pages, keep, from_max, to_max;
  int in_order;            // token j comes from place j, not from place kept[j]
};

// One warp gathers one record: 16 kept tokens of a kv head of a sequence.
template <int D>
__global__ void __launch_bounds__(128) kv4_move_kernel(const Kv4MoveArgs a) {
  using F = Kv4<D>;
  pdl_wait();
  const int lane = threadIdx.x & 31, h = blockIdx.y, seq = blockIdx.z;
  const int n_rec = (a.keep + KV4_TOKENS - 1) / KV4_TOKENS;
  const int rec = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (rec >= n_rec) return;
  const int slot = a.slots[seq];
  if ((unsigned)slot >= (unsigned)a.n_slots) return;
  const size_t head = (size_t)seq * a.nkv + h;
  // lanes 0..15: where the record's tokens come from (as 16-token records and a place in them); -1: no such token, -2: one
  // that no page holds, which goes on as NaN without a weight
  long long src = -1;
  if (lane < KV4_TOKENS) {
    const int j = rec * KV4_TOKENS + lane;
    int from = j < a.keep ? a.kept[head * a.keep + j] : -1;
    if (from >= 0) {
      if (a.in_order) from = j;
      if (a.from_table) {
        const int page = kv4_page(a.from_table + (size_t)slot * a.from_max, from / KV4_PAGE, a.from_max, a.n_pages);
        src = page >= 0 ? ((long long)page * a.nkv + h) * KV4_PAGE + (from & (KV4_PAGE - 1)) : -2;
      } else {
        src = (long long)head * n_rec * KV4_TOKENS + from;
      }
    }
  }
  long long dst;                                          // the record's first token
  if (a.to_table) {
    const int page = kv4_page(a.to_table + (size_t)slot * a.to_max, rec / 4, a.to_max, a.n_pages);
    if (page < 0) return;
    dst = ((long long)page * a.nkv + h) * KV4_PAGE + (rec & 3) * KV4_TOKENS;
  } else {
    dst = ((long long)head * n_rec + rec) * KV4_TOKENS;
  }
  uint8_t* to = a.to + (size_t)(dst / KV4_TOKENS) * F::RECORD;
  // keys: rows as they are; values: chunks of 4 NG bytes, moved where their order turns; pairs
  constexpr int KC = F::ROW / 16, VC = 8;
  uint4 k[KV4_TOKENS * KC / 32];
#pragma unroll
  for (int u = 0; u < KV4_TOKENS * KC / 32; ++u) {
    const int c = u * 32 + lane, tok = c / KC;
    const long long sp = __shfl_sync(0xffffffffu, src, tok);
    k[u] = make_uint4(0, 0, 0, 0);
    if (sp >= 0)
      k[u] = *reinterpret_cast<const uint4*>(a.from + (size_t)(sp / KV4_TOKENS) * F::RECORD + (sp & 15) * F::ROW + (c % KC) * 16);
  }
  uint32_t v[KV4_TOKENS * VC / 32][F::NG];
#pragma unroll
  for (int u = 0; u < KV4_TOKENS * VC / 32; ++u) {
    const int c = u * 32 + lane, tok = c / VC;
    const long long sp = __shfl_sync(0xffffffffu, src, tok);
#pragma unroll
    for (int g = 0; g < F::NG; ++g) v[u][g] = 0u;
    if (sp >= 0) {
      const int from_tok = sp & 15, chunk = (c % VC) ^ F::turn(tok) ^ F::turn(from_tok);
      const uint32_t* p = reinterpret_cast<const uint32_t*>(a.from + (size_t)(sp / KV4_TOKENS) * F::RECORD + F::V_OFF +
                                                            from_tok * F::ROW) + chunk * F::NG;
#pragma unroll
      for (int g = 0; g < F::NG; ++g) v[u][g] = p[g];
    }
  }
  uint32_t pr[2 * F::NG];
#pragma unroll
  for (int g = 0; g < 2 * F::NG; ++g) pr[g] = 0x7fff7fffu;       // (NaN, NaN)
  float w = 0.f;
  if (src >= 0) {
    const uint32_t* p = reinterpret_cast<const uint32_t*>(a.from + (size_t)(src / KV4_TOKENS) * F::RECORD + F::PAIR_OFF +
                                                          (src & 15) * F::PAIR);
#pragma unroll
    for (int g = 0; g < 2 * F::NG; ++g) pr[g] = p[g];
    w = a.w_from[src];
  }
#pragma unroll
  for (int u = 0; u < KV4_TOKENS * KC / 32; ++u) {
    const int c = u * 32 + lane, tok = c / KC;
    if (__shfl_sync(0xffffffffu, src, tok) != -1) *reinterpret_cast<uint4*>(to + tok * F::ROW + (c % KC) * 16) = k[u];
  }
#pragma unroll
  for (int u = 0; u < KV4_TOKENS * VC / 32; ++u) {
    const int c = u * 32 + lane, tok = c / VC;
    if (__shfl_sync(0xffffffffu, src, tok) != -1) {
      uint32_t* p = reinterpret_cast<uint32_t*>(to + F::V_OFF + tok * F::ROW) + (c % VC) * F::NG;
#pragma unroll
      for (int g = 0; g < F::NG; ++g) p[g] = v[u][g];
    }
  }
  if (src != -1) {
    uint32_t* p = reinterpret_cast<uint32_t*>(to + F::PAIR_OFF + lane * F::PAIR);
#pragma unroll
    for (int g = 0; g < 2 * F::NG; ++g) p[g] = pr[g];
    a.w_to[dst + lane] = w;
  }
}

static int choose(const Kv4ChooseArgs* a, cudaStream_t s) {
  if (a->n_seqs < 0 || a->nkv <= 0 || a->max_pages <= 0 || a->max_pages > 0x7fffffff / KV4_PAGE || a->n_pages <= 0 ||
      a->first < 0 || a->recent < 0 || a->keep <= 0 || a->first > a->keep || a->recent > a->keep - a->first)
    return GB_ERR_BAD_ARG;
  if (a->n_seqs > GB_MAX_GRID_YZ) return GB_ERR_UNSUPPORTED;
  const long long room = (long long)a->max_pages * KV4_PAGE;
  const int held = room < CHOOSE_HELD ? (int)room : CHOOSE_HELD;
  static bool configured[64] = {};     // (the shared-memory size is a property of a kernel on one device)
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev >= 64 || !configured[dev]) {
    e = cudaFuncSetAttribute(kv4_choose_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, CHOOSE_HELD * 4);
    if (e != cudaSuccess) return (int)e;
    if (dev < 64) configured[dev] = true;
  }
  return gb_launch(kv4_choose_kernel, dim3(a->nkv, a->n_seqs), dim3(CHOOSE_THREADS), (size_t)held * 4, s, *a, held);
}

static int move(const Kv4MoveArgs* a, int D, cudaStream_t s) {
  if (a->n_seqs < 0 || a->nkv <= 0 || a->keep <= 0 || a->keep > 0x7fffff00 || !a->from || !a->to || !a->kept ||
      (((uintptr_t)a->from | (uintptr_t)a->to) & 15))
    return GB_ERR_BAD_ARG;
  if (a->nkv > GB_MAX_GRID_YZ || a->n_seqs > GB_MAX_GRID_YZ) return GB_ERR_UNSUPPORTED;
  const int n_rec = (a->keep + KV4_TOKENS - 1) / KV4_TOKENS;
  const dim3 grid((n_rec + 3) / 4, a->nkv, a->n_seqs);
  if (D == 64) return gb_launch(kv4_move_kernel<64>, grid, dim3(128), 0, s, *a);
  if (D == 128) return gb_launch(kv4_move_kernel<128>, grid, dim3(128), 0, s, *a);
  return GB_ERR_UNSUPPORTED;
}

// The choice, then the kept tokens moved: straight to their pages, or (back not null) out of the pages and back.
GB_EXPORT int gb_kv4_evict(const Kv4ChooseArgs* c, const Kv4MoveArgs* out, const Kv4MoveArgs* back, int D, cudaStream_t s) {
  if (c->n_seqs == 0) return 0;
  if (D != 64 && D != 128) return GB_ERR_UNSUPPORTED;
  int rc = choose(c, s);
  if (!rc) rc = move(out, D, s);
  if (!rc && back) rc = move(back, D, s);
  return rc;
}
