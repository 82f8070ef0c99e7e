// Attention of single tokens over the cache in 4 bits (kv4.cuh), in bfloat16 on the tensor cores and in 32 bits, and
// the weights that the cached tokens gather from it.
#include "attn_mma.cuh"   // ScoreCap, add_sink, mma_16816
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
  float* part_o;           // [rows, nq, n_splits, D]   (n_splits > 1)
  float* part_ml;          // [rows, nq, n_splits, 2]
  int* error;
  const float* sinks;      // [nq] one more logit of every head's denominator, or null
  int n_rows, n_seqs, n_slots, nq, nkv, max_pages, n_pages, window, n_splits;
  int keep_first, chunk;
  float scale_log2;
  ScoreCap cap;
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

// ---------------------------------------------------------------- bfloat16, single tokens
template <int D>
struct Kv4Decode {
  static constexpr int WARPS = 4;
  static constexpr int STAGES = 3;
  static constexpr int UNIT = 64;                               // keys of a stage: whole records of one page
  static constexpr int RECORDS = UNIT / KV4_TOKENS;
  static constexpr int STAGE_BYTES = RECORDS * Kv4<D>::RECORD;
  static constexpr int RING = WARPS * STAGES * STAGE_BYTES;
  static constexpr int MERGE = WARPS * 8 * (D + 2) * 4;         // the warps' results, where the ring was
  static constexpr int SMEM = (RING > MERGE ? RING : MERGE) + 128;
};

// The scores of a record's 16 tokens with eight query heads: s[0], s[1] are row r's with heads 2 t, 2 t + 1, s[2], s[3]
// row r + 8's, in units of q . k.  The products see a code c as 1 + c / 16; they start from minus the sum of the
// query's elements, so that they end as the sum of q c / 16, and a group's pair then makes 16 s of it and adds m times
// the query's sum.  (Everything is exact but the 32-bit sums: a bfloat16 query times five bits.)
template <int D>
__device__ __forceinline__ void kv4_scores(const uint32_t (&ka)[D / 32], const uint32_t (&kb)[D / 32], const uint32_t* pa,
                                           const uint32_t* pb, const uint32_t (&q)[D / 32][4],
                                           const float (&qsum)[D / 64][2], float (&s)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] = 0.f;
#pragma unroll
  for (int g = 0; g < D / 64; ++g) {
    float acc[4] = {-qsum[g][0], -qsum[g][1], -qsum[g][0], -qsum[g][1]};
#pragma unroll
    for (int w = 2 * g; w < 2 * g + 2; ++w) {
      const uint32_t a0[4] = {kv4_two<0>(ka[w]), kv4_two<0>(kb[w]), kv4_two<1>(ka[w]), kv4_two<1>(kb[w])};
      mma_16816(acc, a0, q[w][0], q[w][1]);
      const uint32_t a1[4] = {kv4_two<2>(ka[w]), kv4_two<2>(kb[w]), kv4_two<3>(ka[w]), kv4_two<3>(kb[w])};
      mma_16816(acc, a1, q[w][2], q[w][3]);
    }
    const float sa = 16.f * kv4_s(pa[g]), ma = kv4_m(pa[g]), sb = 16.f * kv4_s(pb[g]), mb = kv4_m(pb[g]);
    s[0] += fmaf(sa, acc[0], ma * qsum[g][0]);
    s[1] += fmaf(sa, acc[1], ma * qsum[g][1]);
    s[2] += fmaf(sb, acc[2], mb * qsum[g][0]);
    s[3] += fmaf(sb, acc[3], mb * qsum[g][1]);
  }
}

// This lane's part of eight query heads as the B operand (head lane / 4; words n with n % 4 = lane % 4 of its row) and
// the sums of heads 2 t, 2 t + 1 over the groups.  `row`: the head's D elements, or null (zeros).
template <int D>
__device__ __forceinline__ void kv4_query(const bf16* row, uint32_t (&q)[D / 32][4], float (&qsum)[D / 64][2]) {
  const int lane = threadIdx.x & 31, t = lane & 3;
  float part[D / 64];
#pragma unroll
  for (int g = 0; g < D / 64; ++g) part[g] = 0.f;
#pragma unroll
  for (int w = 0; w < D / 32; ++w) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row) v = *reinterpret_cast<const uint4*>(row + 8 * (4 * w + t));
    q[w][0] = v.x, q[w][1] = v.y, q[w][2] = v.z, q[w][3] = v.w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      part[w / 2] += __uint_as_float(q[w][i] << 16) + __uint_as_float(q[w][i] & 0xffff0000u);
  }
#pragma unroll
  for (int g = 0; g < D / 64; ++g) {
    float x = part[g];
    x += __shfl_xor_sync(0xffffffffu, x, 1);
    x += __shfl_xor_sync(0xffffffffu, x, 2);
    qsum[g][0] = __shfl_sync(0xffffffffu, x, 8 * t);        // head 2 t lies in lanes 4 (2 t) ...
    qsum[g][1] = __shfl_sync(0xffffffffu, x, 8 * t + 4);
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

// Block (split, group of up to eight query heads of one kv head, sequence); every warp takes stretches of 64 keys in
// turn, each through a ring of its own that bulk copies fill, and keeps its own maximum, sum and accumulator: no
// barrier of the block lies in the loop.  For 16 tokens at a time
//   S = K q^T       m16n8k16 products, rows tokens, columns heads (kv4_scores)
//   P = 2^(S c - m) in registers; times the value's s it becomes the B operand of the second product by a transposition
//                   of 8 x 8 numbers among the lanes
//   O += V^T P      rows the head's elements, columns heads
// so the codes go from shared memory straight into operands: a word of them is a load, and a shift and a logical
// operation for every two elements.  Values are seen as 1 + c / 16 too: O's excess is the sum of the rounded P, which
// one more product with ones keeps in step, so nothing is lost to the rounding of P.
template <int D>
__global__ void __launch_bounds__(Kv4Decode<D>::WARPS * 32) kv4_decode_kernel(const Kv4AttnArgs a) {
  using F = Kv4<D>;
  using C = Kv4Decode<D>;
  constexpr int NG = F::NG;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t full[C::WARPS][C::STAGES];
  const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int r = lane >> 2, t = lane & 3;
  const int G = a.nq / a.nkv, hgroups = (G + 7) / 8;
  const int split = blockIdx.x, kvh = blockIdx.y / hgroups, hg = blockIdx.y % hgroups, seq = blockIdx.z;
  const int h0 = kvh * G + hg * 8, heads = min(8, G - hg * 8);
  if (lane == 0) {
    for (int s = 0; s < C::STAGES; ++s) mbar_init(&full[warp][s], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  pdl_wait();
  const int slot = a.slots[seq];
  const bool live = (unsigned)slot < (unsigned)a.n_slots;
  const int pos = live ? a.kv_len[seq] - 1 : -1;
  const Stretches list(pos, C::UNIT, a.window, a.keep_first, a.chunk);
  const int keep = a.window > 0 ? a.keep_first : 0;
  const int per = (list.n + a.n_splits - 1) / a.n_splits;
  const int v_end = min(list.n, (split + 1) * per), v0 = split * per + warp;
  const int* table = a.block_table + (size_t)(live ? slot : 0) * a.max_pages;
  uint8_t* ring = smem + warp * C::STAGES * C::STAGE_BYTES;

  // asks for stretch v (a whole warp calls; one lane asks): true when something comes
  bool lost = false;                                 // a page that there is not: the result is NaN
  auto ask = [&](int v, int stage) {
    const int key0 = list.at(v) * C::UNIT;
    const int page = kv4_page(table, key0 / KV4_PAGE, a.max_pages, a.n_pages);
    if (page < 0) {
      lost = true;
      return false;
    }
    const int records = min(C::RECORDS, (pos - key0) / KV4_TOKENS + 1);
    if (elect_one()) {
      const uint32_t bytes = records * F::RECORD;
      mbar_expect_tx(&full[warp][stage], bytes);
      bulk_load(ring + stage * C::STAGE_BYTES,
                a.pages + (((size_t)page * a.nkv + kvh) * (KV4_PAGE / KV4_TOKENS) + (key0 % KV4_PAGE) / KV4_TOKENS) * F::RECORD,
                bytes, &full[warp][stage]);
    }
    __syncwarp();
    return true;
  };
  uint32_t asked = 0, parity = 0;                    // stages with something on its way; the phase to wait for
#pragma unroll
  for (int s = 0; s < C::STAGES; ++s)
    if (v0 + s * C::WARPS < v_end && ask(v0 + s * C::WARPS, s)) asked |= 1u << s;

  uint32_t q[D / 32][4];
  float qsum[NG][2];
  kv4_query<D>(r < heads ? reinterpret_cast<const bf16*>(a.q) + ((size_t)seq * a.nq + h0 + r) * D : nullptr, q, qsum);

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};   // of heads 2 t, 2 t + 1; l and off: this lane's rows only
  float o[NG][4][4], ones_o[NG][4], off[NG][2];
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    off[g][0] = off[g][1] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ones_o[g][i] = 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) o[g][i][c] = 0.f;
    }
  }
  const bool capped = a.cap.cap_log2 != 0.f;
  const int tok_a = kv4_token(r), k_tok = t, k_tok1 = 4 + (t ^ 1);   // tokens of this lane's rows, of its columns
  const int v_word = (r ^ ((t & 2) << 1)) * NG;
  bool ok = true;

  int stage = 0;
  for (int v = v0; v < v_end; v += C::WARPS) {
    if (asked >> stage & 1) {
      if (!mbar_wait_warp(&full[warp][stage], parity >> stage & 1, nullptr)) { ok = false; break; }
      parity ^= 1u << stage;
      const uint8_t* unit = ring + stage * C::STAGE_BYTES;
      const int key0 = list.at(v) * C::UNIT;
      const int records = min(C::RECORDS, (pos - key0) / KV4_TOKENS + 1);
      const bool edge = key0 < list.lo || key0 + C::UNIT - 1 > pos;
#pragma unroll 1
      for (int rec = 0; rec < records; ++rec) {
        const uint8_t* b = unit + rec * F::RECORD;
        uint32_t ka[D / 32], kb[D / 32], pa[2 * NG], pb[2 * NG];
        load_words(b + tok_a * F::ROW + t * (D / 8), ka);
        load_words(b + (tok_a + 8) * F::ROW + t * (D / 8), kb);
        load_words(b + F::PAIR_OFF + tok_a * F::PAIR, pa);
        load_words(b + F::PAIR_OFF + (tok_a + 8) * F::PAIR, pb);
        uint32_t va[4][NG];
        load_words(b + F::V_OFF + k_tok * F::ROW + v_word * 4, va[0]);
        load_words(b + F::V_OFF + k_tok1 * F::ROW + v_word * 4, va[1]);
        load_words(b + F::V_OFF + (k_tok + 8) * F::ROW + v_word * 4, va[2]);
        load_words(b + F::V_OFF + (k_tok1 + 8) * F::ROW + v_word * 4, va[3]);
        float s[4];
        kv4_scores<D>(ka, kb, pa, pb, q, qsum, s);
        if (capped) {
#pragma unroll
          for (int i = 0; i < 4; ++i) s[i] = capped_log2(s[i] * a.cap.cap_inv, a.cap);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) s[i] *= a.scale_log2;
        }
        bool see_a = true, see_b = true;
        if (edge) {
          const int ja = key0 + rec * KV4_TOKENS + tok_a, jb = ja + 8;
          see_a = ja <= pos && (ja >= list.lo || ja < keep);
          see_b = jb <= pos && (jb >= list.lo || jb < keep);
          if (!see_a) s[0] = s[1] = -INFINITY;
          if (!see_b) s[2] = s[3] = -INFINITY;
        }
        // the base of a head's exponents is raised only when a score has outgrown it by 2^8 (or is the first)
        const float x0 = fmaxf(s[0], s[2]), x1 = fmaxf(s[1], s[3]);
        if (__any_sync(0xffffffffu, x0 > m[0] + 8.f || x1 > m[1] + 8.f)) {
          float n0 = x0, n1 = x1;
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) {
            n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, d));
            n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, d));
          }
          n0 = fmaxf(n0, m[0]), n1 = fmaxf(n1, m[1]);
          const float f0 = m[0] == -INFINITY ? 0.f : exp2_fast(m[0] - n0);
          const float f1 = m[1] == -INFINITY ? 0.f : exp2_fast(m[1] - n1);
          m[0] = n0, m[1] = n1;
          l[0] *= f0, l[1] *= f1;
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            off[g][0] *= f0, off[g][1] *= f1;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              ones_o[g][i] *= (i & 1) ? f1 : f0;
#pragma unroll
              for (int c = 0; c < 4; ++c) o[g][i][c] *= (c & 1) ? f1 : f0;
            }
          }
        }
        const float b0 = m[0] == -INFINITY ? 0.f : m[0], b1 = m[1] == -INFINITY ? 0.f : m[1];
        float p[4] = {exp2_fast(s[0] - b0), exp2_fast(s[1] - b1), exp2_fast(s[2] - b0), exp2_fast(s[3] - b1)};
        l[0] += p[0] + p[2];
        l[1] += p[1] + p[3];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          // (a token that is not seen may have a pair of another life, NaN too: it is taken as 0)
          const float sa = see_a ? kv4_s(pa[NG + g]) : 0.f, sb = see_b ? kv4_s(pb[NG + g]) : 0.f;
          const float ma = see_a ? kv4_m(pa[NG + g]) : 0.f, mb = see_b ? kv4_m(pb[NG + g]) : 0.f;
          off[g][0] += fmaf(p[0], ma, p[2] * mb);
          off[g][1] += fmaf(p[1], ma, p[3] * mb);
          const uint32_t p0 = transposed8x8(pack2(p[0] * sa, p[1] * sa));
          const uint32_t p1 = transposed8x8(pack2(p[2] * sb, p[3] * sb));
          const uint32_t one[4] = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
          mma_16816(ones_o[g], one, p0, p1);
          const uint32_t ya = __byte_perm(va[0][g], va[1][g], 0x5410), za = __byte_perm(va[0][g], va[1][g], 0x7632);
          const uint32_t yb = __byte_perm(va[2][g], va[3][g], 0x5410), zb = __byte_perm(va[2][g], va[3][g], 0x7632);
          const uint32_t e0[4] = {kv4_two<0>(ya), kv4_two<0>(za), kv4_two<0>(yb), kv4_two<0>(zb)};
          mma_16816(o[g][0], e0, p0, p1);
          const uint32_t e1[4] = {kv4_two<1>(ya), kv4_two<1>(za), kv4_two<1>(yb), kv4_two<1>(zb)};
          mma_16816(o[g][1], e1, p0, p1);
          const uint32_t e2[4] = {kv4_two<2>(ya), kv4_two<2>(za), kv4_two<2>(yb), kv4_two<2>(zb)};
          mma_16816(o[g][2], e2, p0, p1);
          const uint32_t e3[4] = {kv4_two<3>(ya), kv4_two<3>(za), kv4_two<3>(yb), kv4_two<3>(zb)};
          mma_16816(o[g][3], e3, p0, p1);
        }
      }
      asked &= ~(1u << stage);
      __syncwarp();                                    // all lanes have read the stage
    }
    const int next = v + C::STAGES * C::WARPS;
    if (next < v_end && ask(next, stage)) asked |= 1u << stage;
    stage = stage + 1 == C::STAGES ? 0 : stage + 1;
  }
  if (!ok) {                                           // gave up: wait for what is still on its way, say so, go on to
    for (int s = 0; s < C::STAGES; ++s)                // the block's barriers (the result is void)
      if (asked >> s & 1) mbar_wait_warp(&full[warp][s], parity >> s & 1, nullptr);
    if (lane == 0) atomicCAS(a.error, 0, GB_ERR_KV4_TIMEOUT);
  }
  pdl_launch_dependents();
  if (lost) m[0] = m[1] = 0.f, l[0] = l[1] = __int_as_float(0x7fffffff);

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
  __syncthreads();                                     // every warp has left its ring: the results go there
  float* red_o = reinterpret_cast<float*>(smem);       // [warps][8][D]
  float* red_ml = red_o + C::WARPS * 8 * D;            // [warps][8][2]
#pragma unroll
  for (int g = 0; g < NG; ++g)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        red_o[((size_t)warp * 8 + 2 * t + (c & 1)) * D + g * 64 + 8 * r + 2 * i + (c >> 1)] =
            fmaf(16.f, o[g][i][c] - ones_o[g][c & 1], off[g][c & 1]);
  if (r == 0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      red_ml[(warp * 8 + 2 * t + i) * 2] = m[i];
      red_ml[(warp * 8 + 2 * t + i) * 2 + 1] = l[i];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * D; i += C::WARPS * 32) {
    const int head = i / D, d = i % D;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < C::WARPS; ++w) M = fmaxf(M, red_ml[(w * 8 + head) * 2]);
    float L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < C::WARPS; ++w) {
      const float mw = red_ml[(w * 8 + head) * 2];
      const float f = mw == -INFINITY ? 0.f : exp2f(mw - M);
      L += red_ml[(w * 8 + head) * 2 + 1] * f;
      O += red_o[((size_t)w * 8 + head) * D + d] * f;
    }
    const size_t row = (size_t)seq * a.nq + h0 + head;
    if (a.n_splits == 1) {
      if (a.sinks && live && a.sinks[h0 + head] != -INFINITY) O *= add_sink(a.sinks[h0 + head], M, L);
      reinterpret_cast<bf16*>(a.out)[row * D + d] = __float2bfloat16(L != 0.f ? O / L : 0.f);
      if (a.lse && d == 0) a.lse[row] = L != 0.f ? (M + log2f(L)) * 0.6931471805599453f : -INFINITY;
    } else {
      a.part_o[(row * a.n_splits + split) * D + d] = O;
      if (d == 0) *reinterpret_cast<float2*>(a.part_ml + (row * a.n_splits + split) * 2) = make_float2(M, L);
    }
  }
}

// out[row] from the partial results of the splits, in their order; one block a (row, head).
template <typename T>
__global__ void kv4_merge_kernel(const Kv4AttnArgs a, int D) {
  pdl_wait();
  const size_t row = blockIdx.x, p0 = row * a.n_splits;
  const int seq = a.row_seq ? a.row_seq[row / a.nq] : (int)(row / a.nq);
  const bool live = (unsigned)seq < (unsigned)a.n_seqs && (unsigned)a.slots[seq] < (unsigned)a.n_slots;
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + p0;
  float M = -INFINITY;
  for (int s = 0; s < a.n_splits; ++s) M = fmaxf(M, ml[s].x);
  const float sink = a.sinks && live ? a.sinks[row % a.nq] * 1.4426950408889634f : -INFINITY;
  M = fmaxf(M, sink);
  const int d = threadIdx.x;
  float L = sink == -INFINITY ? 0.f : exp2f(sink - M), O = 0.f;
  for (int s = 0; s < a.n_splits; ++s) {
    const float2 v = ml[s];
    if (v.x == -INFINITY) continue;
    const float f = exp2f(v.x - M);
    L += v.y * f;
    O += a.part_o[(p0 + s) * D + d] * f;
  }
  reinterpret_cast<T*>(a.out)[row * D + d] = from_f32<T>(L != 0.f ? O / L : 0.f);
  if (a.lse && d == 0) a.lse[row] = L != 0.f ? (M + log2f(L)) * 0.6931471805599453f : -INFINITY;
}

// ---------------------------------------------------------------- 32 bits
#define KV4_F32_WARPS 4
#define KV4_F32_HEADS 4

// One row, up to four query heads of a kv head and a split of the keys a block; a warp takes 32 keys at a time.
// Scores: a lane has a key and multiplies its elements with the queries, which lie in shared memory.  Values: half a
// warp has a key, a lane the elements of one word (D 64: a quarter).  32-bit throughout; the scores see a code as
// 1 + c / 16 (its bits at the top of the mantissa) and start from minus the query's sum, as in kv4_scores.
template <int D>
__global__ void __launch_bounds__(KV4_F32_WARPS * 32) kv4_f32_kernel(const Kv4AttnArgs a) {
  using F = Kv4<D>;
  constexpr int NG = F::NG, HC = KV4_F32_HEADS, W = D / 8, LANES = W, KEYS = 32 / LANES;
  __shared__ __align__(16) float q_s[HC][D];
  __shared__ float qsum_s[HC][NG];
  __shared__ float p_s[KV4_F32_WARPS][32][HC];            // P of the warp's keys
  __shared__ float red_o[KV4_F32_WARPS][HC][D];
  __shared__ float red_ml[KV4_F32_WARPS][HC][2];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int G = a.nq / a.nkv, hgroups = (G + HC - 1) / HC;
  const int row = blockIdx.x / a.n_splits, split = blockIdx.x % a.n_splits;
  const int kvh = blockIdx.y / hgroups, hg = blockIdx.y % hgroups;
  const int h0 = kvh * G + hg * HC, heads = min(HC, G - hg * HC);
  const int seq = a.row_seq ? a.row_seq[row] : row;
  const bool known = (unsigned)seq < (unsigned)a.n_seqs;
  const int slot = known ? a.slots[seq] : -1;
  const bool live = (unsigned)slot < (unsigned)a.n_slots;
  const int behind = a.row_seq && known ? a.cu_q[seq + 1] - 1 - row : 0;    // rows of the sequence behind this one
  const int pos = live ? a.kv_len[seq] - 1 - behind : -1;
  const Stretches list(pos, 32, a.window, a.keep_first, a.chunk);
  const int keep = a.window > 0 ? a.keep_first : 0;
  const int per = (list.n + a.n_splits - 1) / a.n_splits;
  const int v_end = min(list.n, (split + 1) * per);
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
  for (int v = split * per + warp; v < v_end; v += KV4_F32_WARPS) {
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
        for (int h = 0; h < HC; ++h) acc[h] = -qsum_s[h][g];
#pragma unroll
        for (int n = 8 * g; n < 8 * g + 8; ++n) {
          const uint32_t w = codes[F::key_word(n)];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int at = ((e & 1) << 4) + ((e >> 1) << 2);
            const float c = __uint_as_float(((at < 19 ? w << (19 - at) : w >> (at - 19)) & 0x00780000u) | 0x3f800000u);
#pragma unroll
            for (int h = 0; h < HC; ++h) acc[h] = fmaf(q_s[h][8 * n + e], c, acc[h]);
          }
        }
        const float sc = 16.f * kv4_s(pair[g]), mn = kv4_m(pair[g]);
#pragma unroll
        for (int h = 0; h < HC; ++h) s[h] += fmaf(sc, acc[h], mn * qsum_s[h][g]);
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
      float p[HC];
      bool any = false;
#pragma unroll
      for (int h = 0; h < HC; ++h) {
        p[h] = p_s[warp][j][h];
        any = any || p[h] != 0.f;
      }
      if (!any) continue;                                  // (not seen, or of no weight: whatever its pair holds)
      const uint32_t pr = reinterpret_cast<const uint32_t*>(rec + F::PAIR_OFF + tok * F::PAIR)[NG + group];
      const uint32_t w = reinterpret_cast<const uint32_t*>(rec + F::V_OFF + tok * F::ROW)[F::value_word(word, tok)];
      const float sc = kv4_s(pr), mn = kv4_m(pr);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = fmaf(sc, (float)kv4_code(w, e), mn);
#pragma unroll
        for (int h = 0; h < HC; ++h) o[h][e] = fmaf(p[h], x, o[h][e]);
      }
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
    const size_t at = (size_t)row * a.nq + h0 + head;
    if (a.n_splits == 1) {
      if (a.sinks && live && a.sinks[h0 + head] != -INFINITY) O *= add_sink(a.sinks[h0 + head], M, L);
      reinterpret_cast<float*>(a.out)[at * D + d] = L != 0.f ? O / L : 0.f;
      if (a.lse && d == 0) a.lse[at] = L != 0.f ? (M + log2f(L)) * 0.6931471805599453f : -INFINITY;
    } else {
      a.part_o[(at * a.n_splits + split) * D + d] = O;
      if (d == 0) *reinterpret_cast<float2*>(a.part_ml + (at * a.n_splits + split) * 2) = make_float2(M, L);
    }
  }
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

// weights[j] += the sum over the sequence's last rows and the kv head's query heads of 2^(s_j c - lse): a warp owns a
// record of a kv head of a sequence, takes its keys into registers once and adds row after row, head after head, in
// that order; nobody else touches the record's weights.
template <int D>
__global__ void __launch_bounds__(WEIGH_WARPS * 32) kv4_weigh_kernel(const Kv4WeighArgs a) {
  using F = Kv4<D>;
  constexpr int NG = F::NG;
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, t = lane & 3;
  const int kvh = blockIdx.y, seq = blockIdx.z, G = a.nq / a.nkv;
  const int slot = a.slots[seq];
  if ((unsigned)slot >= (unsigned)a.n_slots) return;
  const int row1 = a.cu_q[seq + 1], row_first = a.cu_q[seq];
  const int row0 = a.last > 0 ? max(row_first, row1 - a.last) : row_first;
  if (row0 >= row1 || row_first < 0 || row1 > a.n_rows) return;
  const int len = a.kv_len[seq];
  const int pos0 = len - (row1 - row0);                          // the position of row0
  const int* table = a.block_table + (size_t)slot * a.max_pages;
  const int lowest = first_key(max(pos0, 0), a.window, a.chunk);  // no row sees a key below it but for the kept ones
  const int keep = a.window > 0 ? a.keep_first : 0;
  const int records = (len + KV4_TOKENS - 1) / KV4_TOKENS;
  for (int rec = blockIdx.x * WEIGH_WARPS + warp; rec < records; rec += gridDim.x * WEIGH_WARPS) {
    const int key0 = rec * KV4_TOKENS;
    if (key0 + KV4_TOKENS <= lowest && key0 >= keep) continue;
    const int page = kv4_page(table, key0 / KV4_PAGE, a.max_pages, a.n_pages);
    if (page < 0) continue;
    const size_t at = (size_t)page * a.nkv + kvh;
    const uint8_t* b = a.pages + (at * (KV4_PAGE / KV4_TOKENS) + (rec & 3)) * F::RECORD;
    const int tok = kv4_token(r), ja = key0 + tok, jb = ja + 8;
    uint32_t ka[D / 32], kb[D / 32], pa[2 * NG], pb[2 * NG];
    load_words(b + tok * F::ROW + t * (D / 8), ka);
    load_words(b + (tok + 8) * F::ROW + t * (D / 8), kb);
    load_words(b + F::PAIR_OFF + tok * F::PAIR, pa);
    load_words(b + F::PAIR_OFF + (tok + 8) * F::PAIR, pb);
    float wa = 0.f, wb = 0.f;
    for (int row = row0; row < row1; ++row) {
      const int pos = pos0 + row - row0, lo = first_key(max(pos, 0), a.window, a.chunk);
      const bool see_a = ja <= pos && (ja >= lo || ja < keep), see_b = jb <= pos && (jb >= lo || jb < keep);
      if (!__any_sync(0xffffffffu, see_a || see_b)) continue;
      for (int hc = 0; hc < G; hc += 8) {
        const int h0 = kvh * G + hc, heads = min(8, G - hc);
        uint32_t q[D / 32][4];
        float qsum[NG][2], s[4];
        kv4_query<D>(r < heads ? a.q + ((size_t)row * a.nq + h0 + r) * D : nullptr, q, qsum);
        kv4_scores<D>(ka, kb, pa, pb, q, qsum, s);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float lse = 2 * t + i < heads ? a.lse[(size_t)row * a.nq + h0 + 2 * t + i] * 1.4426950408889634f : -INFINITY;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const float x = s[2 * half + i];
            const float y = a.cap.cap_log2 != 0.f ? capped_log2(x * a.cap.cap_inv, a.cap) : x * a.scale_log2;
            if (lse != -INFINITY && (half ? see_b : see_a)) (half ? wb : wa) += exp2f(y - lse);
          }
        }
      }
    }
    wa += __shfl_xor_sync(0xffffffffu, wa, 1), wb += __shfl_xor_sync(0xffffffffu, wb, 1);
    wa += __shfl_xor_sync(0xffffffffu, wa, 2), wb += __shfl_xor_sync(0xffffffffu, wb, 2);
    float* w = a.weights + at * KV4_PAGE + (key0 & (KV4_PAGE - 1));
    if (t == 0 && ja < len) w[tok] += wa;
    if (t == 1 && jb < len) w[tok + 8] += wb;
  }
}

// ---------------------------------------------------------------- entry points
static int checked(const Kv4AttnArgs* a, int D) {
  if (D != 64 && D != 128) return GB_ERR_UNSUPPORTED;
  if (!a->q || !a->pages || !a->out || !a->block_table || !a->slots || !a->kv_len || a->n_rows < 0 || a->n_seqs < 0 ||
      a->nq <= 0 || a->nkv <= 0 || a->nq % a->nkv || a->max_pages <= 0 || a->n_pages <= 0 || a->n_slots < 0 ||
      a->n_splits <= 0 || a->chunk < 0 || a->window < 0 || a->keep_first < 0)
    return GB_ERR_BAD_ARG;
  if (a->n_splits > 1 && (!a->part_o || !a->part_ml)) return GB_ERR_BAD_ARG;
  if (((uintptr_t)a->q | (uintptr_t)a->pages) & 15) return GB_ERR_BAD_ARG;
  return 0;
}

// The shared-memory size is a property of a kernel on one device; it is set once on each.
template <int D>
static int decode(const Kv4AttnArgs& a, cudaStream_t s) {
  static bool configured[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev >= 64 || !configured[dev]) {
    e = cudaFuncSetAttribute(kv4_decode_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Kv4Decode<D>::SMEM);
    if (e != cudaSuccess) return (int)e;
    if (dev < 64) configured[dev] = true;
  }
  const int hgroups = (a.nq / a.nkv + 7) / 8;
  if ((long long)a.nkv * hgroups > 65535 || a.n_seqs > 65535) return GB_ERR_UNSUPPORTED;
  int rc = gb_launch(kv4_decode_kernel<D>, dim3(a.n_splits, a.nkv * hgroups, a.n_seqs), dim3(Kv4Decode<D>::WARPS * 32),
                     Kv4Decode<D>::SMEM, s, a);
  if (rc || a.n_splits == 1) return rc;
  return gb_launch(kv4_merge_kernel<bf16>, dim3((unsigned)(a.n_rows * a.nq)), dim3(D), 0, s, a, D);
}

GB_EXPORT int gb_attn_kv4_decode(const Kv4AttnArgs* a, int D, cudaStream_t s) {
  const int rc = checked(a, D);
  if (rc) return rc;
  if (!a->error || a->n_rows != a->n_seqs || a->row_seq) return GB_ERR_BAD_ARG;
  if ((long long)a->n_rows * a->nq > 0x7fffffffll) return GB_ERR_UNSUPPORTED;
  if (a->n_rows == 0) return 0;
  return D == 64 ? decode<64>(*a, s) : decode<128>(*a, s);
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
  const dim3 grid((unsigned)(a->n_rows * a->n_splits), a->nkv * hgroups);
  rc = D == 64 ? gb_launch(kv4_f32_kernel<64>, grid, dim3(KV4_F32_WARPS * 32), 0, s, *a)
               : gb_launch(kv4_f32_kernel<128>, grid, dim3(KV4_F32_WARPS * 32), 0, s, *a);
  if (rc || a->n_splits == 1) return rc;
  return gb_launch(kv4_merge_kernel<float>, dim3((unsigned)(a->n_rows * a->nq)), dim3(D), 0, s, *a, D);
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
