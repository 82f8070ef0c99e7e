// Attention of single tokens over the cache in 4 bits (kv4.cuh), in bfloat16 on the tensor cores and in 32 bits, and
// the weights that the cached tokens gather from it.
#include <cuda_fp16.h>

#include "attn_mma.cuh"   // ScoreCap, add_sink
#include "kv4.cuh"
#include "tc_common.cuh"  // mbarriers with bounded waits

#define GB_ERR_KV4_TIMEOUT 141

struct Kv4AttnArgs {
  const void* q;           // [rows, nq, D]
  const uint8_t* pages;    // [n_pages, nkv, 4, record]
  const int* block_table;  // [n_slots, max_pages]
  const int* slots;        // [n_seqs]
  const int* kv_len;       // [n_seqs]
  const int* row_seq;      // [rows]: the sequence of a row, or null: row i is sequence i's only one
  const int* cu_q;         // [n_seqs + 1]
  void* out;               // [rows, nq, D]
  float* lse;              // [rows, nq] or null
  float* part_o;           // [parts, heads of a group, D]   (n_splits > 1 and no clusters; see Kv4AttnArgs::part)
  float* part_ml;          // [parts, heads of a group, 2]
  int2* pieces;            // [rows, nkv * groups of heads]: how many parts a pair of row and group has, and its first
  int* error;
  const float* sinks;      // [nq] one more logit of every head's denominator, or null
  int n_rows, n_seqs, n_slots, nq, nkv, max_pages, n_pages, window, n_splits;
  int per;                 // stretches of 32 keys of a split; shared out: that a block takes at least
  int shared;              // 1: the blocks share the stretches out evenly; 2: a pair's splits are a cluster that merges them
  int keep_first, chunk;
  float scale_log2;
  ScoreCap cap;
  // The first part of a pair whose first piece block `block` has.  Blocks that share the stretches out go through the pairs
  // in their order, so that the sum of a block's number and a pair's is another one for every part, and there are no more
  // parts than blocks and pairs: with a place for every split that the bound of the lengths allows, 64 sequences of up to
  // 32,768 keys with 64 heads of 64 on 8 took 68 MB for what now has 2.3.
  __device__ __forceinline__ int part(int pair, int block) const { return shared == 1 ? block + pair : pair * n_splits; }
};

__device__ __forceinline__ float exp2_fast(float x) {   // 2^x, one instruction of the special unit; 2^-inf = 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The stretches of `unit` keys that a query at `pos` reads: with kept first keys those that hold some come first in
// the list, then the window's (the chunk's, or all).
struct Stretches {
  int lo, n_kept, first, n;
  __device__ __forceinline__ Stretches(int pos, int unit, int window, int keep_first, int chunk) {
    lo = first_key(pos, window, chunk);
    const int keep = window > 0 ? keep_first : 0;
    first = lo / unit;
    n_kept = min((min(keep, lo) + unit - 1) / unit, first);
    n = pos < 0 ? 0 : n_kept + pos / unit - first + 1;
  }
  __device__ __forceinline__ int at(int v) const { return v < n_kept ? v : first + v - n_kept; }
};

// The position of row t among its sequence's keys (-1 with no keys), and whether the row is of a sequence at all.
__device__ __forceinline__ bool find_row(const Kv4AttnArgs& a, int t, int& pos) {
  const int seq = a.row_seq ? a.row_seq[t] : t;
  pos = -1;
  if ((unsigned)seq >= (unsigned)a.n_seqs || (unsigned)a.slots[seq] >= (unsigned)a.n_slots) return false;
  pos = a.kv_len[seq] - 1 - (a.row_seq ? a.cu_q[seq + 1] - 1 - t : 0);
  pos = min(pos, a.max_pages * KV4_PAGE);             // (the first place that there is not: it makes the row NaN)
  return true;
}

// ---------------------------------------------------------------- bfloat16, single tokens
#define KV4_SHARED_SEQS 256      // the most sequences whose stretches are shared out (their counts lie beside four rings an SM)

// What beginning and ending a pair's part costs a block, in stretches: every pair counts as so many more, which come in
// front of its own.  (A part more took a block 5.5 us where its stretches took 0.55 each.  60 sequences of up to 4,096
// keys, 200 of up to 1,200, us: counted as none 58.5 and 73.0, six 53.7 and 64.2, ten 53.6 and 63.4, twenty 54.9 and 65.5.)
#define KV4_PART_COST 10
__device__ __forceinline__ int part_stretches(int n) { return n > 0 ? n + KV4_PART_COST : 0; }

// before[i]: the stretches of the sequences in front of i (of one pair of each), their parts' cost included.  Returns how
// many a block takes.  For a whole block of 128 threads.
__device__ __forceinline__ unsigned share_out(const Kv4AttnArgs& a, int unit, int groups, int* before) {
  __shared__ int warp_sums[4];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, each = (a.n_seqs + 127) / 128;
  int mine = 0;
  for (int i = tid * each; i < min(a.n_seqs, (tid + 1) * each); ++i) {
    int pos;
    find_row(a, i, pos);
    mine += part_stretches(Stretches(pos, unit, a.window, a.keep_first, a.chunk).n);
  }
  int sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int below = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += below;
  }
  if (lane == 31) warp_sums[warp] = sum;
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w == warp) sum += all;
    all += warp_sums[w];
  }
  int here = sum - mine;
  for (int i = tid * each; i < min(a.n_seqs, (tid + 1) * each); ++i) {
    int pos;
    find_row(a, i, pos);
    before[i] = here;
    here += part_stretches(Stretches(pos, unit, a.window, a.keep_first, a.chunk).n);
  }
  if (tid == 0) before[a.n_seqs] = all;
  __syncthreads();
  return max((unsigned)a.per, ((unsigned)all * groups + gridDim.x - 1) / gridDim.x);
}

// The sequence that stretch x (of one pair of each sequence) belongs to: the last with before <= x that has any.
__device__ __forceinline__ int find_stretch(const int* before, int n_seqs, unsigned x) {
  int lo = 0, hi = n_seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if ((unsigned)before[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The row of a sequence without keys: zeros (its sink has all the weight, where there is one).
__device__ __forceinline__ void empty_row(const Kv4AttnArgs& a, int seq, int groups, int D) {
  int pos;
  const bool live = find_row(a, seq, pos);
  for (int i = threadIdx.x; i < a.nq * D; i += blockDim.x) reinterpret_cast<bf16*>(a.out)[(size_t)seq * a.nq * D + i] = __float2bfloat16(0.f);
  if (a.lse)
    for (int i = threadIdx.x; i < a.nq; i += blockDim.x)
      a.lse[(size_t)seq * a.nq + i] = live && a.sinks ? a.sinks[i] : -INFINITY;
  for (int i = threadIdx.x; i < groups; i += blockDim.x) a.pieces[(size_t)seq * groups + i] = make_int2(1, 0);
}

template <int D>
struct Kv4Decode {
  static constexpr int WARPS = 4;
  static constexpr int STAGES = 2;                              // (two: the code that gives up knows)
  static constexpr int UNIT = 32;                               // keys of a stage: whole records of one page
  static constexpr int RECORDS = UNIT / KV4_TOKENS;
  static constexpr int STAGE_BYTES = RECORDS * Kv4<D>::RECORD;
  static constexpr int RING = WARPS * STAGES * STAGE_BYTES;
  // The warps' results: 8 heads each, a head's elements in the order (word's element, lane group) under a pitch that
  // puts a store's 32 lanes into 32 banks.
  static constexpr int PITCH = D + 4;
  static constexpr int MERGE = WARPS * 8 * (PITCH + 3) * 4 + 64;
  static constexpr int SMEM = RING + MERGE + 128;
};

// The least score there is (minus infinity would make a NaN of a difference), and the largest power of two that P s is
// multiplied by: P of up to 2^8 times it is a number.
#define KV4_NO_BASE -3e38f
#define KV4_DOWN_MOST 118
__device__ __forceinline__ float kv4_power(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // 2^e

__device__ __forceinline__ __half2 as_half2(uint32_t x) { return *reinterpret_cast<__half2*>(&x); }
__device__ __forceinline__ uint32_t as_u32(__half2 x) { return *reinterpret_cast<uint32_t*>(&x); }

// The eight codes of a word less 8, as four registers of two half-precision numbers (elements 2 i and 2 i + 1; exact).
// A nibble in the low bits of 1024's mantissa is 1024 + c, in the next four 1024 + 16 c, so that a word takes one shift
// and four logical operations, and the multiply-adds that take the rest off run beside them in the other pipe.  (The
// logical pipe has half the rate and is the busiest of these kernels: as bfloat16 numbers, 1 + c / 16, a word takes eight of it.)
// `magic` is 1024 in both halves, from kv4_magic(): an instruction takes one constant, and with two of them the compiler
// makes two instructions of every one of these (144 logical operations a record were counted, then 84; 64 are these masks).
#define KV4_1024 0x64006400u
__device__ __forceinline__ uint32_t kv4_magic(int not_negative) { return KV4_1024 ^ (uint32_t)(not_negative >> 31); }
template <uint32_t MASK>
__device__ __forceinline__ __half2 kv4_nibbles(uint32_t w, uint32_t magic) {
  uint32_t x;                                          // (w & MASK) | magic
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(x) : "r"(w), "n"(MASK), "r"(magic));
  return as_half2(x);
}
__device__ __forceinline__ void kv4_codes(uint32_t w, uint32_t magic, uint32_t (&x)[4]) {
  const __half2 low = __floats2half2_rn(-1032.f, -1032.f), high = __floats2half2_rn(-72.f, -72.f);
  const __half2 sixteenth = __floats2half2_rn(0.0625f, 0.0625f);
  const uint32_t v = w >> 8;
  x[0] = as_u32(__hadd2(kv4_nibbles<0x000f000fu>(w, magic), low));
  x[1] = as_u32(__hfma2(kv4_nibbles<0x00f000f0u>(w, magic), sixteenth, high));
  x[2] = as_u32(__hadd2(kv4_nibbles<0x000f000fu>(v, magic), low));
  x[3] = as_u32(__hfma2(kv4_nibbles<0x00f000f0u>(v, magic), sixteenth, high));
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight query heads as the B operand of the scores: this lane's part of head lane / 4 (words n with n % 4 = lane % 4 of
// its row) in half precision, divided by a power of two that brings the head's largest element into [1, 2): a bfloat16
// element then loses nothing, but for those 2^-15 of the largest and below, which keep 2^-25 of it.  Of heads 2 t and
// 2 t + 1: the sums over the groups (divided too) and the power of two.
template <int D>
struct Kv4Query {
  uint32_t q[D / 32][4];
  float sum[D / 64][2], back[2];
  __device__ __forceinline__ void load(const bf16* row) {       // null: zeros
    const int t = threadIdx.x & 3;
    float x[D / 32][8], top = 0.f;
#pragma unroll
    for (int w = 0; w < D / 32; ++w) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (row) v = *reinterpret_cast<const uint4*>(row + 8 * (4 * w + t));
      const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[w][2 * i] = __uint_as_float(u[i] << 16), x[w][2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        top = fmaxf(top, fmaxf(fabsf(x[w][2 * i]), fabsf(x[w][2 * i + 1])));
      }
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // 2^e <= top, within what a float's inverse can be
    const int e = min(max((int)(__float_as_uint(top) >> 23), 1), 253);
    const float down = __uint_as_float((uint32_t)(254 - e) << 23), up = __uint_as_float((uint32_t)e << 23);
    float part[D / 64];
#pragma unroll
    for (int g = 0; g < D / 64; ++g) part[g] = 0.f;
#pragma unroll
    for (int w = 0; w < D / 32; ++w)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __half2 h = __floats2half2_rn(x[w][2 * i] * down, x[w][2 * i + 1] * down);
        q[w][i] = as_u32(h);
        part[w / 2] += x[w][2 * i] * down + x[w][2 * i + 1] * down;
      }
#pragma unroll
    for (int g = 0; g < D / 64; ++g) {
      float s = part[g];
      s += __shfl_xor_sync(0xffffffffu, s, 1);
      s += __shfl_xor_sync(0xffffffffu, s, 2);
      sum[g][0] = __shfl_sync(0xffffffffu, s, 8 * t);           // head 2 t lies in lanes 4 (2 t) ...
      sum[g][1] = __shfl_sync(0xffffffffu, s, 8 * t + 4);
    }
    back[0] = __shfl_sync(0xffffffffu, up, 8 * t);
    back[1] = __shfl_sync(0xffffffffu, up, 8 * t + 4);
  }
};

// The scores of a record's 16 tokens with eight query heads: s[0], s[1] are row r's with heads 2 t, 2 t + 1, s[2], s[3]
// row r + 8's, in units of q . k over the heads' powers of two.  Products of a half-precision query and codes less 8
// are exact, their sums 32-bit; a group's pair makes s of them and adds m + 8 s times the query's sum.
template <int D>
__device__ __forceinline__ void kv4_scores(const uint32_t (&ka)[D / 32], const uint32_t (&kb)[D / 32], const uint32_t* pa,
                                           const uint32_t* pb, const Kv4Query<D>& q, uint32_t magic, float (&s)[4]) {
#pragma unroll
  for (int g = 0; g < D / 64; ++g) {
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 2 * g; w < 2 * g + 2; ++w) {
      uint32_t xa[4], xb[4];
      kv4_codes(ka[w], magic, xa);
      kv4_codes(kb[w], magic, xb);
      mma_f16(acc, xa[0], xb[0], xa[1], xb[1], q.q[w][0], q.q[w][1]);
      mma_f16(acc, xa[2], xb[2], xa[3], xb[3], q.q[w][2], q.q[w][3]);
    }
    const float sa = kv4_s(pa[g]), ma = fmaf(8.f, sa, kv4_m(pa[g])), sb = kv4_s(pb[g]), mb = fmaf(8.f, sb, kv4_m(pb[g]));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float m = i < 2 ? ma : mb, x = i < 2 ? sa : sb;
      s[i] = g == 0 ? m * q.sum[g][i & 1] : fmaf(m, q.sum[g][i & 1], s[i]);
      s[i] = fmaf(x, acc[i], s[i]);
    }
  }
}

template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    static_assert(N == 1, "one, two or four words");
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

__device__ __forceinline__ uint32_t transposed8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, void* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// The blocks share out the stretches of 32 keys of all pairs (sequence, group of up to eight query heads of one kv head)
// evenly, in the order of the pairs: a block has one run of them, which may end inside a pair and go on in the next, so
// sequences of unequal lengths leave no SM waiting.  (With a fixed number of keys a block the SMs were through with 60
// sequences of 700 to 4,096 keys after 59 to 105 thousand cycles.)  Where the splits fit the GPU at once they are fixed
// instead, a block each, and up to eight of a pair are a cluster that puts its results together; with one split a block
// has a whole pair.
// Of a run's part of a pair every warp takes stretches in turn, each through a ring of its own that bulk copies fill,
// and keeps its own maximum, sum and accumulator: no barrier of the block lies in the loop.  For the two records of a
// stretch
//   S = K q^T       m16n8k16 products, rows tokens, columns heads (kv4_scores)
//   P = 2^(S c - m) in registers; times the value's s it becomes the B operand of the second product by a transposition
//                   of 8 x 8 numbers among the lanes
//   O += V^T P      rows the head's elements, columns heads
// so the codes go from shared memory straight into operands.  P s is half-precision, in units of a power of two for each
// head and group of 64 elements: the largest P s that there was when the unit was chosen, by which a value's s may then be
// exceeded 2^6 times before it is chosen again.  The base of the exponents keeps P below 2^8, so P s stays below 2^15 units,
// and what it loses at the other end is below 2^-25 of one.  (Units by the largest s alone, whatever its token was paid, were
// 1 us faster on the case below, 4 % with many short sequences, and lost all of the others' values beside one 10^9 times as
// large.)  Values are their codes less 8, so the rounding of P (2^-11) meets elements around the middle of their range;
// m + 8 s times P is summed in 32 bits.
// What bounds it: nothing alone.  60 sequences of up to 4,096 keys, 32 heads of 128 on 8, take 52.2 us: 172 MB at 3.3 TB/s
// of 6.45 (26.7 us at the memory's rate).  A record of 16 tokens of a head takes a warp 409 instructions, some 290 of which
// are its own arithmetic (64 logical operations and 64 half-precision ones unpack 4,096 codes, 16 are products): 27 us if
// every scheduler issued on every cycle, and four warps a scheduler issue on 61 % of them, with the logical pipe busy for
// 46 %.  The rest is waiting inside a warp (scores, exponentials and second product of a stretch follow one another),
// blocks that end at different times (the SMs were at work for 64 to 92 thousand cycles, 84 on average) and the merge.
// Three blocks an SM with 168 registers and no spills are no faster.
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A number in the shared memory of block `rank` of the cluster, at the same place as here.
__device__ __forceinline__ float cluster_read(const float* here, int rank) {
  uint32_t at;
  float x;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(here)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(at) : "memory");
  return x;
}

// Element d of a row's head from its maximum, sum and accumulator: the sink joins, and the quotient is stored.
template <typename T>
__device__ __forceinline__ void finish_row(const Kv4AttnArgs& a, int t, bool live, int h, int d, int D, float M, float L,
                                           float O) {
  const size_t row = (size_t)t * a.nq + h;
  if (a.sinks && live && a.sinks[h] != -INFINITY) O *= add_sink(a.sinks[h], M, L);
  reinterpret_cast<T*>(a.out)[row * D + d] = from_f32<T>(L != 0.f ? O / L : 0.f);
  if (a.lse && d == 0) a.lse[row] = L != 0.f ? (M + log2f(L)) * 0.6931471805599453f : -INFINITY;
}

// The splits of some heads of a row are a cluster: each has left its sums [heads][D] and (maximum, sum)s in its shared
// memory and finishes a share of the elements from all of them.
template <typename T>
__device__ __forceinline__ void finish_cluster(const Kv4AttnArgs& a, const float* sums, const float2* ml, int t, bool live,
                                               int h0, int heads, int D, int rank) {
  cluster_barrier();
  const int n = a.n_splits;
  for (int i = threadIdx.x * n + rank; i < heads * D; i += blockDim.x * n) {
    const int h = i / D, d = i % D;
    float M = -INFINITY, L = 0.f, O = 0.f;
    for (int c = 0; c < n; ++c) M = fmaxf(M, cluster_read(&ml[h].x, c));
    for (int c = 0; c < n; ++c) {
      const float mc = cluster_read(&ml[h].x, c), f = mc == -INFINITY ? 0.f : exp2f(mc - M);
      L += cluster_read(&ml[h].y, c) * f;
      O += cluster_read(sums + i, c) * f;
    }
    finish_row<T>(a, t, live, h0 + h, d, D, M, L, O);
  }
  cluster_barrier();                                   // (nobody leaves while its sums are read)
}

// A block's part of a pair, for all its threads.
struct Kv4Part {
  int seq, group, piece, n_pieces;
};

// BOUNDED: there is a window or chunks, so the list of stretches may have a gap and a first key.
template <int D, bool BOUNDED>
__global__ void __launch_bounds__(Kv4Decode<D>::WARPS * 32, 4) kv4_decode_kernel(const Kv4AttnArgs a) {
  using F = Kv4<D>;
  using C = Kv4Decode<D>;
  constexpr int NG = F::NG, NR = C::RECORDS;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t full[C::WARPS][C::STAGES];
  __shared__ int before[KV4_SHARED_SEQS + 1];
  __shared__ Kv4Part part_s[2];
  const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int r = lane >> 2, t = lane & 3;
  const int G = a.nq / a.nkv, hgroups = (G + 7) / 8;
  const int groups = a.nkv * hgroups;
  if (lane == 0) {
    for (int s = 0; s < C::STAGES; ++s) mbar_init(&full[warp][s], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  pdl_wait();
  const int keep = a.window > 0 ? a.keep_first : 0;
  uint8_t* ring = smem + warp * C::STAGES * C::STAGE_BYTES;
  const uint32_t magic = kv4_magic(a.n_seqs);
  uint32_t turn = 0;                                 // stretches that this warp has taken: its stage and its phase follow
  bool ok = true;

  // this block's run [at, end) of the list of all stretches; before[i]: those of one pair of each sequence in front of i
  unsigned at = 0, end = 0, run = 1;
  int seq_next = blockIdx.x / (groups * a.n_splits);
  bool more = true;
  if (a.shared == 1) {
    run = share_out(a, C::UNIT, groups, before);
    at = run * blockIdx.x;
    end = min(at + run, (unsigned)before[a.n_seqs] * groups);
    for (int i = blockIdx.x; i < a.n_seqs; i += gridDim.x)      // sequences without keys have nobody else
      if (before[i + 1] == before[i]) empty_row(a, i, groups, D);
    seq_next = find_stretch(before, a.n_seqs, at / groups);
    if (at < end) {
      // (a run that lies in a pair's cost, but for its end, has nothing to do)
      const unsigned first = (unsigned)before[seq_next] * groups, whole = (unsigned)(before[seq_next + 1] - before[seq_next]);
      more = end > first + (at - first) / whole * whole + KV4_PART_COST;
    } else {
      more = false;
    }
  }
  if (!more) return;

  // The part that is worked on: its sequence's last position and first key, this warp's `mine` stretches from v on (every
  // fourth of the block's).  begin() finds the block's next part and asks for its first stretches; the results of the
  // part before are put together while they come.
  int pos = 0, lo = 0, v = 0, mine = 0, gap_at = 0, gap = 0;
  const int* table = nullptr;
  const uint8_t* head = nullptr;                     // the kv head's records of page 0
  bool lost = false;                                 // a page that there is not: the result is NaN
  int pages = 0;                                     // lane i: the page of the i-th of 32 stretches
  const size_t page_bytes = (size_t)a.nkv * (KV4_PAGE / KV4_TOKENS) * F::RECORD;
  auto first_of = [&](int u) { return (BOUNDED && u >= gap_at ? u + gap : u) * C::UNIT; };
  // looks up the pages of stretches k .. k + 31 of this warp's
  auto look_up = [&](int k) {
    pages = 0;
    if (k + lane < mine) {
      pages = kv4_page(table, first_of(v + (k + lane) * C::WARPS) / KV4_PAGE, a.max_pages, a.n_pages);
      lost = lost || pages < 0;
      pages = max(pages, 0);
    }
  };
  // asks for stretch k of this warp's (the whole warp calls; one lane asks)
  auto ask = [&](int k, uint32_t at_turn) {
    const int page = __shfl_sync(0xffffffffu, pages, k & 31), key0 = first_of(v + k * C::WARPS);
    const uint32_t stage = at_turn % C::STAGES;
    if (elect_one()) {
      const uint32_t bytes = min(NR, (pos - key0) / KV4_TOKENS + 1) * F::RECORD;
      mbar_expect_tx(&full[warp][stage], bytes);
      bulk_load(ring + stage * C::STAGE_BYTES, head + page * page_bytes + key0 % KV4_PAGE / KV4_TOKENS * F::RECORD, bytes,
                &full[warp][stage]);
    }
    __syncwarp();
  };
  int turn_of = 0;                                   // which of part_s has the part that is worked on
  auto begin = [&]() {
    Kv4Part part;
    part.seq = seq_next;
    const bool live = find_row(a, part.seq, pos);
    const int slot = live ? a.slots[part.seq] : 0;
    const Stretches list(pos, C::UNIT, BOUNDED ? a.window : 0, BOUNDED ? a.keep_first : 0, BOUNDED ? a.chunk : 0);
    int v_begin, v_end;
    if (a.shared == 1) {
      // the pair's own stretches are [pair, pair + n) of the list, behind its cost
      const unsigned first = (unsigned)before[part.seq] * groups, n = (unsigned)list.n, whole = n + KV4_PART_COST;
      part.group = (int)((at - first) / whole);
      const unsigned pair = first + part.group * whole + KV4_PART_COST, piece0 = pair / run;
      v_begin = (int)(max(at, pair) - pair);
      v_end = (int)min(n, end - pair);
      part.piece = (int)(blockIdx.x - piece0);
      part.n_pieces = (int)((pair + n - 1) / run - piece0) + 1;
      at = pair + v_end;
      more = at < end && end - at > KV4_PART_COST;      // (and not only a next pair's cost)
      if (at == (unsigned)before[part.seq + 1] * groups && more)
        do ++seq_next; while (before[seq_next + 1] == before[seq_next]);      // (there is one with keys)
    } else {
      part.group = blockIdx.x / a.n_splits % groups, part.piece = blockIdx.x % a.n_splits;
      part.n_pieces = a.n_splits > 1 ? (list.n + a.per - 1) / a.per : 1;
      v_begin = part.piece * a.per;
      v_end = a.n_splits > 1 ? min(list.n, v_begin + a.per) : list.n;
      more = false;
    }
    if (threadIdx.x == 0) part_s[turn_of] = part;
    v = v_begin + warp;
    mine = ok ? max(0, (v_end - v + C::WARPS - 1) / C::WARPS) : 0;
    lo = list.lo, gap_at = list.n_kept, gap = list.first - list.n_kept;
    table = a.block_table + (size_t)slot * a.max_pages;
    head = a.pages + (size_t)(part.group / hgroups) * (KV4_PAGE / KV4_TOKENS) * F::RECORD;
    lost = a.n_splits > 1 && part.n_pieces > a.n_splits;   // (keys beyond the caller's bound of the lengths)
    look_up(0);
#pragma unroll
    for (int k = 0; k < C::STAGES; ++k)
      if (k < mine) ask(k, turn + k);
    return part;
  };

  const int tok_a = kv4_token(r), k_tok = t, k_tok1 = 4 + (t ^ 1);   // tokens of this lane's rows, of its columns
  const int k_at = tok_a * F::ROW + t * (D / 8), p_at = F::PAIR_OFF + tok_a * F::PAIR;
  const int v_word = (r ^ ((t & 2) << 1)) * NG;
  const int v_at = F::V_OFF + k_tok * F::ROW + v_word * 4, v_at1 = F::V_OFF + k_tok1 * F::ROW + v_word * 4;
  const bool capped = a.cap.cap_log2 != 0.f;
  float* red_o = reinterpret_cast<float*>(smem + C::RING);     // [warps][8][PITCH]
  float* red_ml = red_o + C::WARPS * 8 * C::PITCH;             // [warps][8][2]
  float* red_f = red_ml + C::WARPS * 8 * 2;                    // [warps][8]
  float2* red_h = reinterpret_cast<float2*>(red_f + C::WARPS * 8);     // [8]

  Kv4Part part = begin();
  // (a split without keys has asked for nothing; of a cluster it stays for the others)
  if (a.shared != 2 && part.piece > 0 && part.piece >= part.n_pieces) return;
  for (;;) {
    Kv4Query<D> q;
    {
      const int h = part.group % hgroups * 8 + r;
      q.load(h < G ? reinterpret_cast<const bf16*>(a.q) + ((size_t)part.seq * a.nq + part.group / hgroups * G + h) * D : nullptr);
    }
    const float unit_scale = capped ? a.cap.cap_inv : a.scale_log2;
    const float factor[2] = {unit_scale * q.back[0], unit_scale * q.back[1]};

    // of heads 2 t, 2 t + 1: the base of the exponents (a whole number; KV4_NO_BASE: none yet); the sum of P and of P (m + 8 s)
    // over this lane's rows
    float base[2] = {KV4_NO_BASE, KV4_NO_BASE}, l[2] = {0.f, 0.f};
    float o[NG][4][4], off[NG][2];
    // of a group: the powers of two that P s is multiplied by, and the s beyond which they are looked at again
    float down[NG][2], s_most[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      off[g][0] = off[g][1] = 0.f;
      down[g][0] = down[g][1] = kv4_power(KV4_DOWN_MOST);
      s_most[g] = kv4_power(6 - KV4_DOWN_MOST);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[g][i][c] = 0.f;
    }

#pragma unroll 1
    for (int k = 0; k < mine; ++k, ++turn) {
      {
        const uint32_t stage = turn % C::STAGES;
        if (!mbar_wait_warp(&full[warp][stage], turn / C::STAGES & 1, nullptr)) {
          // gave up: wait for what is still on its way, say so, go on to the block's barriers (the result is void)
          if (k + 1 < mine) mbar_wait_warp(&full[warp][(turn + 1) % C::STAGES], (turn + 1) / C::STAGES & 1, nullptr);
          if (lane == 0) atomicCAS(a.error, 0, GB_ERR_KV4_TIMEOUT);
          ok = false;
          break;
        }
        const uint8_t* unit = ring + stage * C::STAGE_BYTES;
        const int key0 = first_of(v + k * C::WARPS);
        float s[NR][4];
        uint32_t vp[NR][2][NG];                      // the values' pairs of this lane's two rows
#pragma unroll
        for (int u = 0; u < NR; ++u) {
          const uint8_t* b = unit + u * F::RECORD;
          uint32_t ka[D / 32], kb[D / 32], pa[2 * NG], pb[2 * NG];
          load_words(b + k_at, ka);
          load_words(b + k_at + 8 * F::ROW, kb);
          load_words(b + p_at, pa);
          load_words(b + p_at + 8 * F::PAIR, pb);
          kv4_scores<D>(ka, kb, pa, pb, q, magic, s[u]);
#pragma unroll
          for (int g = 0; g < NG; ++g) vp[u][0][g] = pa[NG + g], vp[u][1][g] = pb[NG + g];
#pragma unroll
          for (int i = 0; i < 4; ++i) s[u][i] *= factor[i & 1];
        }
        if (capped) {
#pragma unroll
          for (int u = 0; u < NR; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[u][i] = capped_log2(s[u][i], a.cap);
        }
        if ((BOUNDED && key0 < lo) || key0 + C::UNIT - 1 > pos) {
          // (a token that is not seen may have codes and a pair of another life, or of none: its score is -inf and its
          // pair, which may be NaN, is taken as 0)
#pragma unroll
          for (int u = 0; u < NR; ++u)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const int j = key0 + u * KV4_TOKENS + tok_a + half * 8;
              if (!(j <= pos && (!BOUNDED || j >= lo || j < keep))) {
                s[u][2 * half] = s[u][2 * half + 1] = -INFINITY;
#pragma unroll
                for (int g = 0; g < NG; ++g) vp[u][half][g] = 0u;
              }
            }
        }
        // The base of a head's exponents is raised only when a score has outgrown it by 2^8 (or is the first), by a whole
        // number, and the unit of P s, 1 / down, is looked at again then and when an s is beyond those met so far: it becomes
        // the largest P s that there was or is, so that neither a large value without weight nor one that lost its weight
        // takes bits from the others.
        float x[2] = {fmaxf(s[0][0], s[0][2]), fmaxf(s[0][1], s[0][3])};
#pragma unroll
        for (int u = 1; u < NR; ++u) x[0] = fmaxf(x[0], fmaxf(s[u][0], s[u][2])), x[1] = fmaxf(x[1], fmaxf(s[u][1], s[u][3]));
        bool outgrown = x[0] > base[0] + 8.f || x[1] > base[1] + 8.f;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          float sv = 0.f;
#pragma unroll
          for (int u = 0; u < NR; ++u) sv = fmaxf(sv, fmaxf(kv4_s(vp[u][0][g]), kv4_s(vp[u][1][g])));
          outgrown = outgrown || sv > s_most[g];
        }
        if (__any_sync(0xffffffffu, outgrown)) {
          float f[2];
          int steps[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) x[i] = fmaxf(x[i], __shfl_xor_sync(0xffffffffu, x[i], d));
            const float to = fmaxf(base[i], ceilf(x[i])), by = fminf(to - base[i], 1000.f);
            f[i] = exp2_fast(-by), steps[i] = (int)by;
            l[i] *= f[i];
            base[i] = to;
          }
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            float w[2] = {0.f, 0.f};                 // (a NaN has no part)
#pragma unroll
            for (int u = 0; u < NR; ++u)
#pragma unroll
              for (int c = 0; c < 4; ++c)
                w[c & 1] = fmaxf(w[c & 1], exp2_fast(s[u][c] - base[c & 1]) * kv4_s(vp[u][c >> 1][g]));
            // the exponents of both heads' in one word
            uint32_t both = __byte_perm(__float_as_uint(w[0]), __float_as_uint(w[1]), 0x7632);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) both = __vmaxu2(both, __shfl_xor_sync(0xffffffffu, both, d));
            int most = -KV4_DOWN_MOST;
            float change[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              // (the old sums' unit, and the new one: the exponents of their inverses)
              const int was = (int)(__float_as_uint(down[g][i]) >> 23) - 127 + steps[i];
              const int now = min(min(was, KV4_DOWN_MOST), max(127 - (int)(i ? both >> 23 : both >> 7 & 255), -KV4_DOWN_MOST));
              change[i] = kv4_power(max(now - was, -126));
              down[g][i] = kv4_power(now);
              most = max(most, now);
              off[g][i] *= f[i];
            }
            s_most[g] = kv4_power(6 - most);
            if (k > 0) {
#pragma unroll
              for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[g][i][c] *= change[c & 1];
            }
          }
        }
#pragma unroll
        for (int u = 0; u < NR; ++u) {
          const uint8_t* b = unit + u * F::RECORD;
          uint32_t va[4][NG];
          load_words(b + v_at, va[0]);
          load_words(b + v_at1, va[1]);
          load_words(b + v_at + 8 * F::ROW, va[2]);
          load_words(b + v_at1 + 8 * F::ROW, va[3]);
          float p[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) p[i] = exp2_fast(s[u][i] - base[i & 1]);
          l[0] += p[0] + p[2];
          l[1] += p[1] + p[3];
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const float sa = kv4_s(vp[u][0][g]), sb = kv4_s(vp[u][1][g]);
            const float ma = fmaf(8.f, sa, kv4_m(vp[u][0][g])), mb = fmaf(8.f, sb, kv4_m(vp[u][1][g]));
            off[g][0] = fmaf(p[2], mb, fmaf(p[0], ma, off[g][0]));
            off[g][1] = fmaf(p[3], mb, fmaf(p[1], ma, off[g][1]));
            const float d0 = down[g][0], d1 = down[g][1];
            const uint32_t p0 = transposed8x8(as_u32(__floats2half2_rn(p[0] * d0 * sa, p[1] * d1 * sa)));
            const uint32_t p1 = transposed8x8(as_u32(__floats2half2_rn(p[2] * d0 * sb, p[3] * d1 * sb)));
            uint32_t ya[4], za[4], yb[4], zb[4];
            kv4_codes(__byte_perm(va[0][g], va[1][g], 0x5410), magic, ya);
            kv4_codes(__byte_perm(va[0][g], va[1][g], 0x7632), magic, za);
            kv4_codes(__byte_perm(va[2][g], va[3][g], 0x5410), magic, yb);
            kv4_codes(__byte_perm(va[2][g], va[3][g], 0x7632), magic, zb);
#pragma unroll
            for (int i = 0; i < 4; ++i) mma_f16(o[g][i], ya[i], za[i], yb[i], zb[i], p0, p1);
          }
        }
        __syncwarp();                                  // all lanes have read the stage
      }
      const int next = k + C::STAGES;
      if (next < mine) {
        if ((next & 31) == 0) look_up(next);
        ask(next, turn + C::STAGES);
      }
    }
    if (__any_sync(0xffffffffu, lost)) base[0] = base[1] = 0.f, l[0] = l[1] = __int_as_float(0x7fffffff);

    const bool again = more;
    turn_of ^= 1;
    if (again) part = begin();
    else pdl_launch_dependents();

    // the sums over the rows of a head's column, and the accumulator in its own units
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) {
      l[0] += __shfl_xor_sync(0xffffffffu, l[0], d);
      l[1] += __shfl_xor_sync(0xffffffffu, l[1], d);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        off[g][0] += __shfl_xor_sync(0xffffffffu, off[g][0], d);
        off[g][1] += __shfl_xor_sync(0xffffffffu, off[g][1], d);
      }
    }
    float up[NG][2];                                   // 1 / down
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int i = 0; i < 2; ++i) up[g][i] = __uint_as_float((254u << 23) - __float_as_uint(down[g][i]));
    __syncthreads();                                   // every warp has read the results of the part before
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          red_o[(warp * 8 + 2 * t + (c & 1)) * C::PITCH + ((g * 4 + i) * 2 + (c >> 1)) * 8 + r] =
              fmaf(up[g][c & 1], o[g][i][c], off[g][c & 1]);
    if (r == 0) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        red_ml[(warp * 8 + 2 * t + i) * 2] = base[i] == KV4_NO_BASE ? -INFINITY : base[i];
        red_ml[(warp * 8 + 2 * t + i) * 2 + 1] = l[i];
      }
    }
    __syncthreads();
    const Kv4Part done = part_s[turn_of ^ 1];
    const int h0 = done.group / hgroups * G + done.group % hgroups * 8, heads = min(8, G - done.group % hgroups * 8);
    // the warps' share of each head, and the head's maximum and sum
    if (threadIdx.x < 8) {
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int w = 0; w < C::WARPS; ++w) M = fmaxf(M, red_ml[(w * 8 + threadIdx.x) * 2]);
#pragma unroll
      for (int w = 0; w < C::WARPS; ++w) {
        const float mw = red_ml[(w * 8 + threadIdx.x) * 2], f = mw == -INFINITY ? 0.f : exp2f(mw - M);
        L += red_ml[(w * 8 + threadIdx.x) * 2 + 1] * f;
        red_f[w * 8 + threadIdx.x] = f;
      }
      red_h[threadIdx.x] = make_float2(M, L);
    }
    __syncthreads();
    const bool alone = done.n_pieces <= 1;             // the result is final
    const bool live = (unsigned)a.slots[done.seq] < (unsigned)a.n_slots;
    if (a.shared == 2) {
      for (int i = threadIdx.x; i < heads * D; i += C::WARPS * 32) {
        const int h = i / D, d = i % D, place = (d & 64) + (d & 7) * 8 + (d >> 3 & 7);
        float O = 0.f;
#pragma unroll
        for (int w = 0; w < C::WARPS; ++w) O += red_o[(w * 8 + h) * C::PITCH + place] * red_f[w * 8 + h];
        reinterpret_cast<float*>(smem)[i] = O;         // (the ring is done with)
      }
      finish_cluster<bf16>(a, reinterpret_cast<const float*>(smem), red_h, done.seq, live, h0, heads, D, done.piece);
      break;
    }
    const int pair = done.seq * groups + done.group, first = a.part(pair, blockIdx.x - done.piece);
    const size_t row0 = (size_t)(first + done.piece) * min(8, G);
    for (int i = threadIdx.x; i < heads * D; i += C::WARPS * 32) {
      const int h = i / D, d = i % D, place = (d & 64) + (d & 7) * 8 + (d >> 3 & 7);
      float O = 0.f;
#pragma unroll
      for (int w = 0; w < C::WARPS; ++w) O += red_o[(w * 8 + h) * C::PITCH + place] * red_f[w * 8 + h];
      const float2 ml = red_h[h];
      if (alone) {
        finish_row<bf16>(a, done.seq, live, h0 + h, d, D, ml.x, ml.y, O);
      } else {
        a.part_o[(row0 + h) * D + d] = O;
        if (d == 0) *reinterpret_cast<float2*>(a.part_ml + (row0 + h) * 2) = ml;
      }
    }
    if (a.n_splits > 1 && done.piece == 0 && threadIdx.x == 0) a.pieces[pair] = make_int2(done.n_pieces, first);
    if (!again) break;
  }
}

// out[row] from the partial results of its splits, in their order; a warp a (row, head): its lanes take the splits'
// factors first, a split a lane, and then D / 32 elements each through all splits.  Rows of one split are finished
// already.  (With a thread for every element, which took the factors for itself, 60 sequences of up to 4,096 keys took
// 53.6 us with their merging, so 50.9, and two of 32,768 29.9 and 27.8.)
#define MERGE_WARPS 4
template <typename T, int D>
__global__ void __launch_bounds__(32 * MERGE_WARPS) kv4_merge_kernel(const Kv4AttnArgs a, int per_group) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31, G = a.nq / a.nkv, hgroups = (G + per_group - 1) / per_group;
  const long long row = (long long)blockIdx.x * MERGE_WARPS + (threadIdx.x >> 5);
  pdl_wait();                                        // (every block: the next kernel waits for this one only)
  if (row >= (long long)a.n_rows * a.nq) return;
  const int t = (int)(row / a.nq), h = (int)(row % a.nq);
  const int2 parts = a.pieces[(size_t)t * a.nkv * hgroups + h / G * hgroups + h % G / per_group];
  const int n = parts.x, heads = min(per_group, G);
  if (n <= 1) return;
  float x[E];
  float M, L;
  if (n > a.n_splits) {                               // keys beyond the caller's bound: some were left out
    M = L = __int_as_float(0x7fffffff);
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = L;
  } else {
    const size_t p0 = (size_t)parts.y * heads + h % G % per_group;
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + p0;       // (the parts' are `heads` apart)
    const float* po = a.part_o + p0 * D + lane * E;
    const float sk = a.sinks ? a.sinks[h] * 1.4426950408889634f : -INFINITY;
    float2 mine = make_float2(-INFINITY, 0.f);        // of split `lane` of the first 32 (of 32 at a time, below)
    if (lane < n) mine = ml[(size_t)lane * heads];
    M = mine.x;
    for (int s = 32 + lane; s < n; s += 32) M = fmaxf(M, ml[(size_t)s * heads].x);
    M = fmaxf(warp_max(M), sk);
    L = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = 0.f;
    for (int s0 = 0; s0 < n; s0 += 32) {
      if (s0 > 0) mine = s0 + lane < n ? ml[(size_t)(s0 + lane) * heads] : make_float2(-INFINITY, 0.f);
      // (a maximum drops NaN, so a split that saw nothing but NaN has the factor 0 and a sum that is NaN: it has to stay)
      const float f = mine.x == -INFINITY ? 0.f : exp2f(mine.x - M);
      L += mine.y * f;
      const int here = min(32, n - s0);
      // (eight splits' loads on their way at a time; those behind the last have the factor 0)
      for (int s = 0; s < here; s += 8) {
        float v[8][E];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const float* from = po + (size_t)(s0 + min(s + u, here - 1)) * heads * D;
          if constexpr (E == 4) {
            const float4 w = *reinterpret_cast<const float4*>(from);
            v[u][0] = w.x, v[u][1] = w.y, v[u][2] = w.z, v[u][3] = w.w;
          } else {
            const float2 w = *reinterpret_cast<const float2*>(from);
            v[u][0] = w.x, v[u][1] = w.y;
          }
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const float fs = __shfl_sync(0xffffffffu, f, min(s + u, 31));
          // (also where the factor is 0: a sum that is NaN has to stay)
#pragma unroll
          for (int e = 0; e < E; ++e) x[e] = fmaf(v[u][e], fs, x[e]);
        }
      }
    }
    L = warp_sum(L);
    if (sk != -INFINITY) L += exp2f(sk - M);
    const float inv = L != 0.f ? 1.f / L : 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] *= inv;
  }
  T* to = reinterpret_cast<T*>(a.out) + (size_t)row * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) to[e] = from_f32<T>(x[e]);
  if (a.lse && lane == 0) a.lse[row] = L != 0.f ? (M + log2f(L)) * 0.6931471805599453f : -INFINITY;
}

template <typename T>
static int merge(const Kv4AttnArgs& a, int D, int per_group, cudaStream_t s) {
  const long long blocks = ((long long)a.n_rows * a.nq + MERGE_WARPS - 1) / MERGE_WARPS;
  if (D == 64) return gb_launch(kv4_merge_kernel<T, 64>, dim3((unsigned)blocks), dim3(32 * MERGE_WARPS), 0, s, a, per_group);
  return gb_launch(kv4_merge_kernel<T, 128>, dim3((unsigned)blocks), dim3(32 * MERGE_WARPS), 0, s, a, per_group);
}

// ---------------------------------------------------------------- 32 bits
#define KV4_F32_WARPS 4
#define KV4_F32_HEADS 4

// One row, up to four query heads of a kv head and a split of the keys a block; a warp takes 32 keys at a time.
// Scores: a lane has a key and multiplies its elements with the queries, which lie in shared memory.  Values: half a
// warp has a key, a lane the elements of one word (D 64: a quarter).  32-bit throughout; the scores see a code as
// (c - 8) / 16 (its bits at the top of 1's mantissa, less 1.5) and add m + 8 s times the query's sum.
template <int D>
__global__ void __launch_bounds__(KV4_F32_WARPS * 32) kv4_f32_kernel(const Kv4AttnArgs a) {
  using F = Kv4<D>;
  constexpr int NG = F::NG, HC = KV4_F32_HEADS, W = D / 8, LANES = W, KEYS = 32 / LANES;
  __shared__ __align__(16) float q_s[HC][D];
  __shared__ float qsum_s[HC][NG];
  __shared__ float p_s[KV4_F32_WARPS][32][HC];            // P of the warp's keys
  __shared__ float red_o[KV4_F32_WARPS][HC][D];
  __shared__ float red_ml[KV4_F32_WARPS][HC][2];
  __shared__ float2 ml_s[HC];                             // of a split of a cluster
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int G = a.nq / a.nkv, hgroups = (G + HC - 1) / HC;
  const int row = blockIdx.x / a.n_splits, split = blockIdx.x % a.n_splits;
  const int kvh = blockIdx.y / hgroups, hg = blockIdx.y % hgroups;
  const int h0 = kvh * G + hg * HC, heads = min(HC, G - hg * HC);
  int pos;
  const bool live = find_row(a, row, pos);
  const int slot = live ? a.slots[a.row_seq ? a.row_seq[row] : row] : -1;
  const Stretches list(pos, 32, a.window, a.keep_first, a.chunk);
  const int keep = a.window > 0 ? a.keep_first : 0;
  const int v_end = a.n_splits == 1 ? list.n : min(list.n, (split + 1) * a.per);
  if (a.shared != 2 && split > 0 && split * a.per >= list.n) return;
  const bool alone = a.n_splits == 1 || list.n <= a.per;
  const int* table = a.block_table + (size_t)(live ? slot : 0) * a.max_pages;
  for (int i = threadIdx.x; i < HC * D; i += blockDim.x)
    q_s[i / D][i % D] = i / D < heads ? reinterpret_cast<const float*>(a.q)[((size_t)row * a.nq + h0) * D + i] : 0.f;
  __syncthreads();
  for (int i = warp; i < HC * NG; i += KV4_F32_WARPS) {
    const float x = warp_sum(q_s[i / NG][i % NG * 64 + lane] + q_s[i / NG][i % NG * 64 + 32 + lane]);
    if (lane == 0) qsum_s[i / NG][i % NG] = x;
  }
  __syncthreads();
  const bool capped = a.cap.cap_log2 != 0.f;
  float m[HC], l[HC], o[HC][8];
#pragma unroll
  for (int h = 0; h < HC; ++h) {
    m[h] = -INFINITY, l[h] = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[h][e] = 0.f;
  }
  const int word = lane % LANES, half = lane / LANES, group = word / 8;   // this lane's elements of a value
  for (int v = split * a.per + warp; v < v_end; v += KV4_F32_WARPS) {
    const int key0 = list.at(v) * 32, key = key0 + lane;
    const int page = kv4_page(table, key0 / KV4_PAGE, a.max_pages, a.n_pages);
    if (page < 0) {                                        // a page that there is not: the result is NaN
#pragma unroll
      for (int h = 0; h < HC; ++h) m[h] = 0.f, l[h] = __int_as_float(0x7fffffff);
      continue;
    }
    const uint8_t* base = a.pages + (((size_t)page * a.nkv + kvh) * (KV4_PAGE / KV4_TOKENS) + (key0 % KV4_PAGE) / KV4_TOKENS) * F::RECORD;
    const bool see = key <= pos && (key >= list.lo || key < keep);
    float s[HC];
    uint32_t pair[2 * NG];
#pragma unroll
    for (int g = 0; g < 2 * NG; ++g) pair[g] = 0;
#pragma unroll
    for (int h = 0; h < HC; ++h) s[h] = 0.f;
    if (see) {
      const uint8_t* rec = base + (lane / KV4_TOKENS) * F::RECORD;
      const int tok = lane % KV4_TOKENS;
      load_words(rec + F::PAIR_OFF + tok * F::PAIR, pair);
      const uint32_t* codes = reinterpret_cast<const uint32_t*>(rec + tok * F::ROW);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float acc[HC];
#pragma unroll
        for (int h = 0; h < HC; ++h) acc[h] = 0.f;
#pragma unroll
        for (int n = 8 * g; n < 8 * g + 8; ++n) {
          const uint32_t w = codes[F::key_word(n)];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int at = ((e & 1) << 4) + ((e >> 1) << 2);
            const float c = __uint_as_float(((at < 19 ? w << (19 - at) : w >> (at - 19)) & 0x00780000u) | 0x3f800000u) - 1.5f;
#pragma unroll
            for (int h = 0; h < HC; ++h) acc[h] = fmaf(q_s[h][8 * n + e], c, acc[h]);
          }
        }
        const float sc = 16.f * kv4_s(pair[g]), mid = fmaf(0.5f, sc, kv4_m(pair[g]));
#pragma unroll
        for (int h = 0; h < HC; ++h) s[h] += fmaf(sc, acc[h], mid * qsum_s[h][g]);
      }
    }
    __syncwarp();                                          // the warp's P of the last keys has been read
#pragma unroll
    for (int h = 0; h < HC; ++h) {
      float x = capped ? capped_log2(s[h] * a.cap.cap_inv, a.cap) : s[h] * a.scale_log2;
      x = see ? x : -INFINITY;
      const float top = fmaxf(m[h], warp_max(x));
      const float base_m = top == -INFINITY ? 0.f : top;
      const float f = m[h] == -INFINITY ? 0.f : exp2f(m[h] - top);
      const float p = exp2f(x - base_m);
      m[h] = top;
      l[h] = l[h] * f + p;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[h][e] *= f;
      p_s[warp][lane][h] = see ? p : 0.f;
    }
    __syncwarp();
    const int n_keys = min(32, pos - key0 + 1);
    for (int j = half; j < n_keys; j += KEYS) {
      const int tok = j % KV4_TOKENS;
      const uint8_t* rec = base + (j / KV4_TOKENS) * F::RECORD;
      if (key0 + j < list.lo && key0 + j >= keep) continue;     // (not seen: whatever its pair holds)
      float p[HC];
#pragma unroll
      for (int h = 0; h < HC; ++h) p[h] = p_s[warp][j][h];
      const uint32_t pr = reinterpret_cast<const uint32_t*>(rec + F::PAIR_OFF + tok * F::PAIR)[NG + group];
      const uint32_t w = reinterpret_cast<const uint32_t*>(rec + F::V_OFF + tok * F::ROW)[F::value_word(word, tok)];
      float x[8];
      kv4_values(w, pr, x);
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int h = 0; h < HC; ++h) o[h][e] = fmaf(p[h], x[e], o[h][e]);
    }
  }
  pdl_launch_dependents();
#pragma unroll
  for (int h = 0; h < HC; ++h) {
    l[h] = warp_sum(l[h]);
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int d = LANES; d < 32; d <<= 1) o[h][e] += __shfl_xor_sync(0xffffffffu, o[h][e], d);
    if (half == 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) red_o[warp][h][word * 8 + e] = o[h][e];
    }
    if (lane == 0) red_ml[warp][h][0] = m[h], red_ml[warp][h][1] = l[h];
  }
  __syncthreads();
  // keys beyond the caller's bound of the lengths make the row NaN (merged by the second kernel, pieces says so)
  const int pair = row * gridDim.y + blockIdx.y;
  const bool beyond = a.shared == 2 && list.n > a.per * a.n_splits;
  for (int i = threadIdx.x; i < heads * D; i += blockDim.x) {
    const int head = i / D, d = i % D;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < KV4_F32_WARPS; ++w) M = fmaxf(M, red_ml[w][head][0]);
    float L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < KV4_F32_WARPS; ++w) {
      const float mw = red_ml[w][head][0], f = mw == -INFINITY ? 0.f : exp2f(mw - M);
      L += red_ml[w][head][1] * f;
      O += red_o[w][head][d] * f;
    }
    if (a.shared == 2) {
      q_s[head][d] = beyond ? __int_as_float(0x7fffffff) : O;           // (the queries are done with)
      if (d == 0) ml_s[head] = make_float2(beyond ? 0.f : M, L);
    } else if (alone) {
      finish_row<float>(a, row, live, h0 + head, d, D, M, L, O);
    } else {
      const size_t at = ((size_t)pair * a.n_splits + split) * min(HC, G) + head;
      a.part_o[at * D + d] = O;
      if (d == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(M, L);
    }
  }
  if (a.shared == 2) finish_cluster<float>(a, &q_s[0][0], ml_s, row, live, h0, heads, D, split);
  else if (a.n_splits > 1 && split == 0 && threadIdx.x == 0)
    a.pieces[pair] = make_int2(max(1, (list.n + a.per - 1) / a.per), a.part(pair, 0));
}

// ---------------------------------------------------------------- the weights that tokens gather
struct Kv4WeighArgs {
  const bf16* q;           // [rows, nq, D]
  const float* lse;        // [rows, nq]: the natural logarithm of every softmax's sum
  const uint8_t* pages;
  float* weights;          // [n_pages, nkv, 64]
  const int* block_table;
  const int* slots;
  const int* kv_len;
  const int* cu_q;         // [n_seqs + 1]
  int n_rows, n_seqs, n_slots, nq, nkv, max_pages, n_pages, window, keep_first, chunk, last;
  float scale_log2;
  ScoreCap cap;
};

#define WEIGH_WARPS 4
#define WEIGH_RECORDS 2      // of a step

// weights[j] += the sum over the sequence's last rows and the kv head's query heads of 2^(s_j c - lse).  The (row, head)
// pairs are the columns of the products, eight at a time.  A warp takes 32 tokens of one kv head at a time, every
// (WEIGH_WARPS x blocks)th of them, with the keys of the next on their way while it sums this one's; nobody else touches
// these tokens' weights, and the order of the sums is always the same.  More than eight columns: a set after the other,
// the keys read again for each (they come from L2).
template <int D>
__global__ void __launch_bounds__(WEIGH_WARPS * 32, 4) kv4_weigh_kernel(const Kv4WeighArgs a) {
  using F = Kv4<D>;
  constexpr int NG = F::NG, NR = WEIGH_RECORDS, STEP = NR * KV4_TOKENS;
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, t = lane & 3;
  const int kvh = blockIdx.y, seq = blockIdx.z, G = a.nq / a.nkv;
  const int slot = a.slots[seq], len = a.kv_len[seq];
  const int row1 = a.cu_q[seq + 1], row_first = a.cu_q[seq];
  const int steps = (int)min((len + (long long)STEP - 1) / STEP, (long long)a.max_pages * (KV4_PAGE / STEP));
  const int stride = gridDim.x * WEIGH_WARPS, step0 = blockIdx.x * WEIGH_WARPS + warp;
  if ((unsigned)slot >= (unsigned)a.n_slots || step0 >= steps) return;
  const int row0 = a.last > 0 ? max(row_first, row1 - a.last) : row_first;
  if (row0 >= row1 || row_first < 0 || row1 > a.n_rows) return;
  const int pos0 = len - (row1 - row0);                          // the position of row0
  const int* table = a.block_table + (size_t)slot * a.max_pages;
  const int lowest = first_key(max(pos0, 0), a.window, a.chunk);  // no row sees a key below it but for the kept ones
  const int keep = a.window > 0 ? a.keep_first : 0;
  const uint32_t magic = kv4_magic(a.n_seqs);
  const int tok = kv4_token(r), columns = (row1 - row0) * G;
  const bool capped = a.cap.cap_log2 != 0.f, bounded = a.window > 0 || a.chunk > 0;

  uint32_t ka[NR][D / 32], kb[NR][D / 32], pa[NR][NG], pb[NR][NG];
  // the record of the head that step s begins with, or null: nothing to do there
  auto record_of = [&](int s) -> const uint8_t* {
    if (s >= steps || (s * STEP + STEP <= lowest && s * STEP >= keep)) return nullptr;
    const int page = kv4_page(table, s * STEP / KV4_PAGE, a.max_pages, a.n_pages);
    if (page < 0) return nullptr;
    return a.pages + (((size_t)page * a.nkv + kvh) * (KV4_PAGE / KV4_TOKENS) + s * STEP % KV4_PAGE / KV4_TOKENS) * F::RECORD;
  };
  auto load = [&](const uint8_t* b) {
    if (!b) return;
#pragma unroll
    for (int u = 0; u < NR; ++u, b += F::RECORD) {
      load_words(b + tok * F::ROW + t * (D / 8), ka[u]);
      load_words(b + (tok + 8) * F::ROW + t * (D / 8), kb[u]);
      load_words(b + F::PAIR_OFF + tok * F::PAIR, pa[u]);
      load_words(b + F::PAIR_OFF + (tok + 8) * F::PAIR, pb[u]);
    }
  };
  for (int c0 = 0; c0 < columns; c0 += 8) {
    const uint8_t* here = record_of(step0);
    load(here);
    const uint8_t* after = record_of(step0 + stride);
    // column c is head c % G of row c / G; this lane loads the query of column c0 + r and sums columns c0 + 2 t, + 2 t + 1
    Kv4Query<D> q;
    {
      const int c = c0 + r;
      q.load(c < columns ? a.q + ((size_t)(row0 + c / G) * a.nq + kvh * G + c % G) * D : nullptr);
    }
    int last[2], first[2];
    float lse[2], factor[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = c0 + 2 * t + i, row = row0 + c / G;
      last[i] = -1, first[i] = 0, lse[i] = 0.f;
      if (c < columns) {
        lse[i] = a.lse[(size_t)row * a.nq + kvh * G + c % G] * 1.4426950408889634f;
        if (lse[i] != -INFINITY) last[i] = pos0 + row - row0, first[i] = first_key(max(last[i], 0), a.window, a.chunk);
      }
      factor[i] = (capped ? a.cap.cap_inv : a.scale_log2) * q.back[i];
    }
    for (int s = step0; s < steps; s += stride) {
      float sum[NR][2];
#pragma unroll
      for (int u = 0; u < NR; ++u) {
        float x[4];
        if (here) kv4_scores<D>(ka[u], kb[u], pa[u], pb[u], q, magic, x);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int j = s * STEP + u * KV4_TOKENS + tok + half * 8;
          sum[u][half] = 0.f;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float y = x[2 * half + i] * factor[i];
            if (capped) y = capped_log2(y, a.cap);
            const float p = exp2_fast(y - lse[i]);
            if (j <= last[i] && (!bounded || j >= first[i] || j < keep)) sum[u][half] += p;
          }
        }
      }
      const bool done = here != nullptr;
      const int page_at = s * STEP;
      float* w = a.weights;
      if (done) {
        const int page = kv4_page(table, page_at / KV4_PAGE, a.max_pages, a.n_pages);
        w += ((size_t)page * a.nkv + kvh) * KV4_PAGE + page_at % KV4_PAGE;
      }
      here = after;
      load(here);
      after = record_of(s + 2 * stride);
      if (!done) continue;
#pragma unroll
      for (int u = 0; u < NR; ++u)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          sum[u][half] += __shfl_xor_sync(0xffffffffu, sum[u][half], 1);
          sum[u][half] += __shfl_xor_sync(0xffffffffu, sum[u][half], 2);
          // Each lane of a row's four has one of its tokens of the step.  (Added where it lies, without waiting for what
          // is there; this lane alone adds to it, in the order of the sets, so the sum is the same every time.)
          const int j = u * KV4_TOKENS + tok + half * 8;
          if (t == u * 2 + half && page_at + j < len) atomicAdd(w + j, sum[u][half]);
        }
    }
  }
}

// ---------------------------------------------------------------- entry points
static int checked(const Kv4AttnArgs* a, int D) {
  if (D != 64 && D != 128) return GB_ERR_UNSUPPORTED;
  if (!a->q || !a->pages || !a->out || !a->block_table || !a->slots || !a->kv_len || a->n_rows < 0 || a->n_seqs < 0 ||
      a->nq <= 0 || a->nkv <= 0 || a->nq % a->nkv || a->max_pages <= 0 || a->max_pages > 0x1000000 || a->n_pages <= 0 || a->n_slots < 0 ||
      a->n_splits <= 0 || a->per <= 0 || a->chunk < 0 || a->window < 0 || a->keep_first < 0)
    return GB_ERR_BAD_ARG;
  if (a->n_splits > 1 && a->shared != 2 && (!a->part_o || !a->part_ml || !a->pieces)) return GB_ERR_BAD_ARG;
  if (((uintptr_t)a->q | (uintptr_t)a->pages) & 15) return GB_ERR_BAD_ARG;
  return 0;
}

template <int D, bool BOUNDED>
static int decode_launch(const Kv4AttnArgs& a, unsigned grid, cudaStream_t s) {
  static bool configured[64] = {};     // (the shared-memory size is a property of a kernel on one device)
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev >= 64 || !configured[dev]) {
    e = cudaFuncSetAttribute(kv4_decode_kernel<D, BOUNDED>, cudaFuncAttributeMaxDynamicSharedMemorySize, Kv4Decode<D>::SMEM);
    if (e != cudaSuccess) return (int)e;
    if (dev < 64) configured[dev] = true;
  }
  return gb_launch_cluster(kv4_decode_kernel<D, BOUNDED>, dim3(grid), dim3(Kv4Decode<D>::WARPS * 32), Kv4Decode<D>::SMEM, s,
                           a.shared == 2 ? a.n_splits : 1, a);
}

template <int D>
static int decode(const Kv4AttnArgs& a, int blocks, cudaStream_t s) {
  const int hgroups = (a.nq / a.nkv + 7) / 8;
  const long long pairs = (long long)a.nkv * hgroups * a.n_seqs;
  if (pairs * a.n_splits > 0x7fffffffll) return GB_ERR_UNSUPPORTED;
  // (all stretches are counted in 32 bits, and a block's run may reach beyond them)
  if (a.shared == 2 && (a.n_splits < 2 || a.n_splits > 8)) return GB_ERR_BAD_ARG;
  if (a.shared == 1 && (a.n_splits < 2 || a.n_seqs > KV4_SHARED_SEQS || blocks <= 0 ||
                   pairs * (4ll * a.max_pages + 64) + 2ll * blocks * a.per > 0x7fffffffll))
    return GB_ERR_BAD_ARG;
  const unsigned grid = (unsigned)(a.shared == 1 ? blocks : pairs * a.n_splits);
  const int rc = a.window > 0 || a.chunk > 0 ? decode_launch<D, true>(a, grid, s) : decode_launch<D, false>(a, grid, s);
  if (rc || a.n_splits == 1 || a.shared == 2) return rc;
  return merge<bf16>(a, D, 8, s);
}

// `blocks`: how many share the keys out (a->shared 1).
GB_EXPORT int gb_attn_kv4_decode(const Kv4AttnArgs* a, int D, int blocks, cudaStream_t s) {
  const int rc = checked(a, D);
  if (rc) return rc;
  if (!a->error || a->n_rows != a->n_seqs || a->row_seq) return GB_ERR_BAD_ARG;
  if ((long long)a->n_rows * a->nq > 0x7fffffffll) return GB_ERR_UNSUPPORTED;
  if (a->n_rows == 0) return 0;
  return D == 64 ? decode<64>(*a, blocks, s) : decode<128>(*a, blocks, s);
}

GB_EXPORT int gb_attn_kv4_f32(const Kv4AttnArgs* a, int D, cudaStream_t s) {
  int rc = checked(a, D);
  if (rc) return rc;
  if (a->row_seq ? !a->cu_q : a->n_rows != a->n_seqs) return GB_ERR_BAD_ARG;
  const int hgroups = (a->nq / a->nkv + KV4_F32_HEADS - 1) / KV4_F32_HEADS;
  if ((long long)a->n_rows * a->n_splits > 0x7fffffffll || (long long)a->nkv * hgroups > 65535 ||
      (long long)a->n_rows * a->nq > 0x7fffffffll)
    return GB_ERR_UNSUPPORTED;
  if (a->n_rows == 0) return 0;
  if (a->shared && (a->shared != 2 || a->n_splits < 2 || a->n_splits > 8)) return GB_ERR_BAD_ARG;
  const dim3 grid((unsigned)(a->n_rows * a->n_splits), a->nkv * hgroups);
  const int cluster = a->shared == 2 ? a->n_splits : 1;
  rc = D == 64 ? gb_launch_cluster(kv4_f32_kernel<64>, grid, dim3(KV4_F32_WARPS * 32), 0, s, cluster, *a)
               : gb_launch_cluster(kv4_f32_kernel<128>, grid, dim3(KV4_F32_WARPS * 32), 0, s, cluster, *a);
  if (rc || a->n_splits == 1 || cluster > 1) return rc;
  return merge<float>(*a, D, KV4_F32_HEADS, s);
}

// `blocks`: blocks along the keys of every (kv head, sequence).
GB_EXPORT int gb_kv4_weigh(const Kv4WeighArgs* a, int D, int blocks, cudaStream_t s) {
  if (D != 64 && D != 128) return GB_ERR_UNSUPPORTED;
  if (!a->q || !a->lse || !a->pages || !a->weights || !a->block_table || !a->slots || !a->kv_len || !a->cu_q || a->n_rows < 0 ||
      a->n_seqs < 0 || a->nq <= 0 || a->nkv <= 0 || a->nq % a->nkv || a->max_pages <= 0 || a->n_pages <= 0 || a->n_slots < 0 ||
      a->chunk < 0 || a->window < 0 || a->keep_first < 0 || a->last < 0 || blocks <= 0)
    return GB_ERR_BAD_ARG;
  if (((uintptr_t)a->q | (uintptr_t)a->pages) & 15) return GB_ERR_BAD_ARG;
  if (a->nkv > 65535 || a->n_seqs > 65535) return GB_ERR_UNSUPPORTED;
  if (a->n_rows == 0 || a->n_seqs == 0) return 0;
  const dim3 grid(blocks, a->nkv, a->n_seqs);
  if (D == 64) return gb_launch(kv4_weigh_kernel<64>, grid, dim3(WEIGH_WARPS * 32), 0, s, *a);
  return gb_launch(kv4_weigh_kernel<128>, grid, dim3(WEIGH_WARPS * 32), 0, s, *a);
}
