// A cache in 4 bits (kv4.cuh): keys and values written and read back, and tokens dropped by the weights they gathered.
#include "kv4.cuh"

#define GB_MAX_GRID_YZ 65535

struct Kv4RowsArgs {
  const void* kv;          // [T, 2 nkv, D]: what is written, or (out) what is read
  void* out;
  const int* token_seq;    // [T]
  const int* token_pos;    // [T]
  const int* slots;        // [n_seqs]
  const int* block_table;  // [n_slots, max_pages]
  uint8_t* pages;
  float* weights;          // [n_pages, nkv, 64] set to 0 for the tokens written, or null
  int T, n_seqs, n_slots, nkv, max_pages, n_pages;
};

// Where token t of a step lives: its page (-1: nowhere) and its place there.
__device__ __forceinline__ int find_token(const Kv4RowsArgs& a, int t, int& place) {
  const int seq = a.token_seq[t], pos = a.token_pos[t];
  place = pos & (KV4_PAGE - 1);
  if ((unsigned)seq >= (unsigned)a.n_seqs || pos < 0) return -1;
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

// Eight lanes take a group of 64 elements, a word's eight each: the group's range is three exchanges, its codes and
// pair are written straight to their places.  A row of codes (64 bytes at D 128) comes from one warp.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_write_kernel(const Kv4RowsArgs a) {
  using F = Kv4<D>;
  pdl_wait();
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const long long group = i >> 3;
  const int lane8 = i & 7;
  const long long n_groups = (long long)a.T * 2 * a.nkv * F::NG;
  if (group >= n_groups) return;                       // (whole groups of lanes leave)
  const uint32_t mask = 0xffu << (threadIdx.x & 24);
  const int g = group % F::NG;
  const long long row = group / F::NG;
  const int hh = row % (2 * a.nkv), t = row / (2 * a.nkv);
  float x[8];
  load8(reinterpret_cast<const T*>(a.kv) + row * D + g * KV4_GROUP + lane8 * 8, x);
  int place;
  const int page = find_token(a, t, place);
  if (page < 0) return;                                // (the same for the group's lanes)
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
  uint32_t sb = bf16_away(__fdiv_rn(__fsub_rn(hi, m), 15.f));                     // upwards: it is not negative
  const float s = __uint_as_float(sb << 16);
  uint32_t word = 0, pair = (mb << 16) | sb;
  if (!fine || !isfinite(s) || !isfinite(m)) {
    pair = 0x7fff7fffu;                                // NaN, NaN
  } else if (s > 0.f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t c = (uint32_t)__float2int_rn(__fdiv_rn(__fsub_rn(x[e], m), s));
      word |= min(c, 15u) << (((e & 1) << 4) + ((e >> 1) << 2));
    }
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

// The same lanes the other way: a word and its pair in, eight elements out (zeros for a token that is nowhere).
template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4RowsArgs a) {
  using F = Kv4<D>;
  pdl_wait();
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const int n = i % (D / 8);
  const long long row = i / (D / 8);
  if (row >= (long long)a.T * 2 * a.nkv) return;
  const int hh = row % (2 * a.nkv), t = row / (2 * a.nkv);
  int place;
  const int page = find_token(a, t, place);
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (page >= 0) {
    const bool is_v = hh >= a.nkv;
    const int h = is_v ? hh - a.nkv : hh, tok = place & (KV4_TOKENS - 1);
    const uint8_t* rec = a.pages + (((size_t)page * a.nkv + h) * (KV4_PAGE / KV4_TOKENS) + place / KV4_TOKENS) * F::RECORD;
    const uint32_t* codes = reinterpret_cast<const uint32_t*>(rec + (is_v ? F::V_OFF : 0) + tok * F::ROW);
    const uint32_t w = codes[is_v ? F::value_word(n, tok) : F::key_word(n)];
    const uint32_t pair = reinterpret_cast<const uint32_t*>(rec + F::PAIR_OFF + tok * F::PAIR)[(is_v ? F::NG : 0) + n / 8];
    const float s = kv4_s(pair), m = kv4_m(pair);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmaf(s, (float)kv4_code(w, e), m);
  }
  store8(reinterpret_cast<T*>(a.out) + row * D + n * 8, x);
}

template <typename T, int D>
static int launch_rows(const Kv4RowsArgs& a, bool write, cudaStream_t s) {
  const long long threads = (long long)a.T * 2 * a.nkv * (D / 8), blocks = (threads + 255) / 256;
  if (blocks > 0x7fffffffll) return GB_ERR_UNSUPPORTED;
  return gb_launch(write ? kv4_write_kernel<T, D> : kv4_read_kernel<T, D>, dim3((unsigned)blocks), dim3(256), 0, s, a);
}
static int rows(const Kv4RowsArgs* a, int D, int f32, bool write, cudaStream_t s) {
  if (a->T < 0 || a->nkv <= 0 || a->max_pages <= 0 || a->n_pages <= 0 || a->n_seqs < 0 || a->n_slots < 0 || !a->pages)
    return GB_ERR_BAD_ARG;
  if (((uintptr_t)(write ? a->kv : a->out) | (uintptr_t)a->pages) & 15) return GB_ERR_BAD_ARG;
  if (a->T == 0) return 0;
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

// One block chooses for one kv head of one sequence.  The weight of the last token that is kept among the candidates
// is found digit by digit (four passes over eight bits, a histogram each); one more pass in the order of the tokens
// then writes the places of the kept ones, with the first of those that are equal to the last one kept.
__global__ void __launch_bounds__(CHOOSE_THREADS) kv4_choose_kernel(const Kv4ChooseArgs a) {
  __shared__ int hist[256];
  __shared__ int warp_sum_s[2][32];
  __shared__ uint32_t digit_s;
  __shared__ int left_s;
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
  auto weight = [&](int i) -> uint32_t {
    const int page = kv4_page(table, i / KV4_PAGE, a.max_pages, a.n_pages);
    return page < 0 ? 0u : ordered(a.weights[((size_t)page * a.nkv + h) * KV4_PAGE + (i & (KV4_PAGE - 1))]);
  };
  uint32_t last = 0xffffffffu;                          // the weight of the last one kept (nothing is above it)
  int left = 0;                                         // how many of that weight are kept
  if (need > 0) {
    last = 0;
    left = need;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += CHOOSE_THREADS) hist[i] = 0;
      __syncthreads();
      for (int i = c0 + tid; i < c1; i += CHOOSE_THREADS) {
        const uint32_t u = weight(i);
        if (shift == 24 || (u >> (shift + 8)) == (last >> (shift + 8))) atomicAdd(&hist[(u >> shift) & 255], 1);
      }
      __syncthreads();
      if (warp == 0) {                                  // from the largest digit down: the one where `left` runs out
        int above = 0;
        for (int top = 255; top >= 0; top -= 32) {
          const int n = hist[top - lane];
          int sum = n;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
          }
          const uint32_t hit = __ballot_sync(0xffffffffu, above + sum >= left);
          if (hit) {
            const int at = __ffs(hit) - 1;
            const int before = above + __shfl_sync(0xffffffffu, sum - n, at);
            if (lane == 0) digit_s = (uint32_t)(top - at), left_s = left - before;
            break;
          }
          above += __shfl_sync(0xffffffffu, sum, 31);
        }
      }
      __syncthreads();
      last |= digit_s << shift;
      left = left_s;
      __syncthreads();
    }
  }
  int out = 0, equal = 0;                               // kept, and equal to the last, in front of this stretch
  for (int base = 0; base < len; base += CHOOSE_THREADS) {
    const int i = base + tid;
    const bool in = i < len, sure = in && (i < c0 || i >= c1);
    const uint32_t u = in && !sure && need > 0 ? weight(i) : 0u;
    const bool cand = in && !sure && need > 0;
    const bool tie = cand && u == last;
    const uint32_t ties = __ballot_sync(0xffffffffu, tie);
    if (lane == 0) warp_sum_s[0][warp] = __popc(ties);
    __syncthreads();
    int t_before = 0, t_all = 0;
    for (int w = 0; w < CHOOSE_THREADS / 32; ++w) {
      const int n = warp_sum_s[0][w];
      t_before += w < warp ? n : 0;
      t_all += n;
    }
    const int rank = equal + t_before + __popc(ties & ((1u << lane) - 1));
    const bool mine = sure || (cand && (u > last || (tie && rank < left)));
    const uint32_t who = __ballot_sync(0xffffffffu, mine);
    if (lane == 0) warp_sum_s[1][warp] = __popc(who);
    __syncthreads();
    int k_before = 0, k_all = 0;
    for (int w = 0; w < CHOOSE_THREADS / 32; ++w) {
      const int n = warp_sum_s[1][w];
      k_before += w < warp ? n : 0;
      k_all += n;
    }
    if (mine) kept[out + k_before + __popc(who & ((1u << lane) - 1))] = i;
    out += k_all;
    equal += t_all;
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
  // lanes 0..15: where the record's tokens come from (as 16-token records and a place in them), -1: no such token
  long long src = -1;
  if (lane < KV4_TOKENS) {
    const int j = rec * KV4_TOKENS + lane;
    int from = j < a.keep ? a.kept[head * a.keep + j] : -1;
    if (from >= 0) {
      if (a.in_order) from = j;
      if (a.from_table) {
        const int page = kv4_page(a.from_table + (size_t)slot * a.from_max, from / KV4_PAGE, a.from_max, a.n_pages);
        if (page >= 0) src = ((long long)page * a.nkv + h) * KV4_PAGE + (from & (KV4_PAGE - 1));
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
    if (sp >= 0)
      k[u] = *reinterpret_cast<const uint4*>(a.from + (size_t)(sp / KV4_TOKENS) * F::RECORD + (sp & 15) * F::ROW + (c % KC) * 16);
  }
  uint32_t v[KV4_TOKENS * VC / 32][F::NG];
#pragma unroll
  for (int u = 0; u < KV4_TOKENS * VC / 32; ++u) {
    const int c = u * 32 + lane, tok = c / VC;
    const long long sp = __shfl_sync(0xffffffffu, src, tok);
    if (sp >= 0) {
      const int from_tok = sp & 15, chunk = (c % VC) ^ F::turn(tok) ^ F::turn(from_tok);
      const uint32_t* p = reinterpret_cast<const uint32_t*>(a.from + (size_t)(sp / KV4_TOKENS) * F::RECORD + F::V_OFF +
                                                            from_tok * F::ROW) + chunk * F::NG;
#pragma unroll
      for (int g = 0; g < F::NG; ++g) v[u][g] = p[g];
    }
  }
  uint32_t pr[2 * F::NG];
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
    if (__shfl_sync(0xffffffffu, src, tok) >= 0) *reinterpret_cast<uint4*>(to + tok * F::ROW + (c % KC) * 16) = k[u];
  }
#pragma unroll
  for (int u = 0; u < KV4_TOKENS * VC / 32; ++u) {
    const int c = u * 32 + lane, tok = c / VC;
    if (__shfl_sync(0xffffffffu, src, tok) >= 0) {
      uint32_t* p = reinterpret_cast<uint32_t*>(to + F::V_OFF + tok * F::ROW) + (c % VC) * F::NG;
#pragma unroll
      for (int g = 0; g < F::NG; ++g) p[g] = v[u][g];
    }
  }
  if (src >= 0) {
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
  return gb_launch(kv4_choose_kernel, dim3(a->nkv, a->n_seqs), dim3(CHOOSE_THREADS), 0, s, *a);
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
