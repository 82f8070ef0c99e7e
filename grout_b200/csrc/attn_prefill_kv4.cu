// Prompt attention over a cache in 4 bits: the kernel of attn_prefill_tc.cuh with key tiles that warps of its own
// unpack from the records (kv4.cuh) into the swizzled tiles that the tensor cores read.
//
// An element becomes s c + m in one bfloat16 multiply-add, rounded once: the precision that a cache in bfloat16 would
// have stored it with.  A tile's 128 half rows of keys and of values go to the producer warps' lanes one each (two
// each with two warps); a lane's loads for the next tile are under way while it unpacks this one.
#include "attn_prefill_tc.cuh"
#include "kv4.cuh"

struct Kv4Pages {
  struct Params {
    const uint8_t* pages;
    float* lse;              // [n_tokens, nq] or null
    int n_pages, n_slots;
  };
  // Producer warps: beside two query blocks two for heads of 64 (twelve warps, three a scheduler, have 168 registers each)
  // and four for heads of 128 (fourteen have 128, and the softmax spills a few): a prompt of 2,048 tokens, 32 heads of
  // 128, takes 53.8 us with two and 51.0 with four, windowed chunks with heads of 64 48.2 with two and 49.8 with four.
  template <int DS, int G>
  using Config = AtConfig<DS, G, G == 2 ? 2 * DS : 2>;
  __device__ __forceinline__ static constexpr int FULL_ARRIVALS(int warps) { return warps; }
  __device__ __forceinline__ static float* lse(const Params& p) { return p.lse; }
  __device__ __forceinline__ static int slot(const Params& p, int s) { return s < p.n_slots ? s : -1; }
  __device__ __forceinline__ static void before_padding() { pdl_wait(); }
  __device__ __forceinline__ static void prepare(const Params&) {}
  // C tanh(x) log2 e = C log2 e (1 - 2 / (2^(2 x log2 e) + 1)) with the special unit's power and inverse as they are
  // (2^-22 of their size off; an exponent too small gives 0 and an infinite power's inverse is 0, which are the two
  // ends) and two scores to an instruction around them: six sequences' chunks of up to 384 rows, windowed, 20 heads of
  // 64, take 74.2 us, 83.0 with the powers and quotients of the 16-bit kernel, 48.1 without a cap.
  __device__ __forceinline__ static void cap_scores(float (&s)[AT_BN], const ScoreCap& cap) {
    const float in = cap.cap_inv * 2.8853900817779268f;
    const uint64_t in2 = pack_f32x2(in, in), zero2 = pack_f32x2(0.f, 0.f), one2 = pack_f32x2(1.f, 1.f);
    const uint64_t twice2 = pack_f32x2(-2.f * cap.cap_log2, -2.f * cap.cap_log2), top2 = pack_f32x2(cap.cap_log2, cap.cap_log2);
#pragma unroll
    for (int c = 0; c < AT_BN; c += 2) {
      float x0, x1, r0, r1;
      unpack_f32x2(fma_f32x2(pack_f32x2(s[c], s[c + 1]), in2, zero2), x0, x1);
      unpack_f32x2(add_f32x2(pack_f32x2(fast_exp2(x0), fast_exp2(x1)), one2), x0, x1);
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r0) : "f"(x0));
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r1) : "f"(x1));
      unpack_f32x2(fma_f32x2(pack_f32x2(r0, r1), twice2, top2), s[c], s[c + 1]);
    }
  }

  // What a lane needs of a half row of a key and of a value, and whether its token is one that the block sees.
  template <int D>
  struct Half {
    uint32_t k[D / 16], v[D / 16], pair[2 * Kv4<D>::NG];
    bool see, bad;           // bad: no page holds it
  };

  static __device__ __forceinline__ bool wait_warp(void* bar, uint32_t parity, volatile int* abort_flag) {
    if (__all_sync(0xffffffffu, mbar_try(bar, parity))) return true;
    const unsigned long long t0 = now_ns();
#pragma unroll 1
    for (int i = 1;; ++i) {
      __nanosleep(100);
      if (__all_sync(0xffffffffu, mbar_try(bar, parity))) return true;
      if ((i & 31) == 0) {
        const bool stop = *abort_flag || now_ns() - t0 > TC_WAIT_LIMIT_NS;
        if (__any_sync(0xffffffffu, stop)) return __all_sync(0xffffffffu, mbar_try(bar, parity));
      }
    }
  }

  template <int N>
  static __device__ __forceinline__ void load(const uint8_t* p, uint32_t* w) {
    if constexpr (N == 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x, w[1] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const uint4 v = reinterpret_cast<const uint4*>(p)[i / 4];
        w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
      }
    }
  }

  // The eight elements of a word, s c + m: a code in the low bits of 128's mantissa is 128 + c, less 128 it is c, exactly,
  // and the multiply-add rounds once.  `magic` is 128 in both halves, from a register: with two constants an instruction
  // the compiler makes two of it.
  template <int I>
  static __device__ __forceinline__ uint32_t element2(uint32_t w, uint32_t magic, __nv_bfloat162 s, __nv_bfloat162 m) {
    uint32_t x;                                            // (w >> 4 I & 0x000f000f) | magic
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(x) : "r"(w >> (4 * I)), "n"(0x000f000fu), "r"(magic));
    const __nv_bfloat162 c = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&x), __floats2bfloat162_rn(128.f, 128.f));
    const __nv_bfloat162 y = __hfma2(s, c, m);
    return *reinterpret_cast<const uint32_t*>(&y);
  }
  static __device__ __forceinline__ void unpack8(uint32_t addr, uint32_t w, uint32_t magic, __nv_bfloat162 s, __nv_bfloat162 m) {
    sts128(addr, element2<0>(w, magic, s, m), element2<1>(w, magic, s, m), element2<2>(w, magic, s, m),
           element2<3>(w, magic, s, m));
  }

  template <int DS, int G>
  __device__ __forceinline__ static void produce(const Params& p, const AttnTcArgs& a, const AtTiles& b, int who) {
    using Cfg = Config<DS, G>;
    constexpr int D = 64 * DS, STAGES = Cfg::STAGES, NG = Kv4<D>::NG;
    constexpr int EACH = 2 * AT_BN / (32 * Cfg::PRODUCERS);          // half rows of a lane
    using F = Kv4<D>;
    const int lane = threadIdx.x & 31;
    const uint32_t magic = 0x43004300u ^ (uint32_t)(a.n_seqs >> 31);
    Half<D> next[EACH];
    auto ask = [&](int j) {
      const int tile = b.tile(j);
      const int page = kv4_page(b.table, tile, a.max_pages, p.n_pages);
#pragma unroll
      for (int u = 0; u < EACH; ++u) {
        const int item = (u * Cfg::PRODUCERS + who) * 32 + lane, row = item >> 1, half = item & 1;
        const int key = tile * AT_BN + row, tok = row & (KV4_TOKENS - 1);
        next[u].see = key <= b.hi && (key >= b.lo || key < b.keep);
        next[u].bad = page < 0;
        if (next[u].see && page >= 0) {
          const uint8_t* rec = p.pages + (((size_t)page * a.nkv + b.kvh) * (AT_BN / KV4_TOKENS) + row / KV4_TOKENS) * F::RECORD;
          load<D / 16>(rec + tok * F::ROW + half * (F::ROW / 2), next[u].k);
          load<D / 16>(rec + F::V_OFF + tok * F::ROW + half * (F::ROW / 2), next[u].v);
          load<2 * NG>(rec + F::PAIR_OFF + tok * F::PAIR, next[u].pair);
        }
      }
    };
    if (b.n_tiles > 0) ask(0);
    for (int j = 0; j < b.n_tiles; ++j) {
      Half<D> now[EACH];
#pragma unroll
      for (int u = 0; u < EACH; ++u) now[u] = next[u];
      if (j + 1 < b.n_tiles) ask(j + 1);
      const int s = j % STAGES;
      const uint32_t par = (((uint32_t)(j / STAGES)) & 1) ^ 1;
      bool freed = j - STAGES >= b.n_a || wait_warp(&b.kv_empty[s], par, b.abort_flag);
      freed = freed && (j - STAGES >= b.n_b || wait_warp(&b.kv_empty[STAGES + s], par, b.abort_flag));
      if (!freed) {
        if (lane == 0) {
          if (!*b.abort_flag) atomicCAS(a.error, 0, GB_ERR_AT_TIMEOUT);
          *b.abort_flag = 1;
        }
        break;
      }
      const uint32_t st = smem_u32(b.kv_s + (size_t)s * Cfg::KV_BYTES);
#pragma unroll
      for (int u = 0; u < EACH; ++u) {
        const int item = (u * Cfg::PRODUCERS + who) * 32 + lane, row = item >> 1, half = item & 1;
        const uint32_t krow = st + row * 128, vrow = krow + DS * Cfg::SUB_BYTES, swz = row & 7;
        // A token that no row of the block sees is zeros, whatever its place in the pool holds: its probability is 0,
        // but 0 times a NaN would still be one.  For the same reason a value that is NaN (its pair is) goes in as
        // zeros and makes its key NaN instead, so that the rows that see it, and no others, come out as NaN.
        bool poison = now[u].see && now[u].bad;
        uint32_t kp[NG], vp[NG];
        const bool real = now[u].see && !now[u].bad;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          kp[g] = real ? now[u].pair[g] : 0u;
          vp[g] = real ? now[u].pair[NG + g] : 0u;
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const float s = kv4_s(vp[g]), m = kv4_m(vp[g]);
          if (!(fabsf(s) <= 3.4e38f && fabsf(m) <= 3.4e38f)) poison = true;
        }
        __nv_bfloat162 ks[NG], km[NG], vs[NG], vm[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          if (poison) kp[g] = 0x7fff7fffu, vp[g] = 0u;
          const float s1 = kv4_s(kp[g]), m1 = kv4_m(kp[g]), s2 = kv4_s(vp[g]), m2 = kv4_m(vp[g]);
          ks[g] = __floats2bfloat162_rn(s1, s1), km[g] = __floats2bfloat162_rn(m1, m1);
          vs[g] = __floats2bfloat162_rn(s2, s2), vm[g] = __floats2bfloat162_rn(m2, m2);
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          // word i of a key's half row: lane group t = 2 half + i / (D / 32), word t + 4 w of the head.  (The second
          // half takes its words two by two in the other order: the chunks that eight lanes store at once then lie
          // in different banks.)
          constexpr int W = D / 32;
          const int w = (i % W) ^ half, t = 2 * half + i / W;
          const int g = w / 2, chunk = (w & 1) * 4 + t;
          const uint32_t word = half ? now[u].k[i ^ 1] : now[u].k[i];
          unpack8(krow + g * Cfg::SUB_BYTES + ((uint32_t)(chunk ^ swz) << 4), real ? word : 0u, magic, ks[(i % W) / 2], km[(i % W) / 2]);
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const int g = i % NG, chunk = (4 * half + i / NG) ^ F::turn(row);
          unpack8(vrow + g * Cfg::SUB_BYTES + ((uint32_t)(chunk ^ swz) << 4), real && !poison ? now[u].v[i] : 0u, magic, vs[g], vm[g]);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // visible to the tensor core
      __syncwarp();
      mbar_arrive_if(&b.kv_full[s], lane == 0);
    }
    pdl_launch_dependents();
  }
};

template <int DS, int G>
static int launch(const Kv4Pages::Params& pages, const bf16* q, const AttnTcArgs& a, cudaStream_t s) {
  using Cfg = Kv4Pages::Config<DS, G>;
  static bool configured[64] = {};     // (the shared-memory size is a property of a kernel on one device)
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev >= 64 || !configured[dev]) {
    e = cudaFuncSetAttribute(attn_prefill_tc_kernel<DS, G, Kv4Pages>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg::SMEM);
    if (e != cudaSuccess) return (int)e;
    if (dev < 64) configured[dev] = true;
  }
  return gb_launch(attn_prefill_tc_kernel<DS, G, Kv4Pages>, dim3(a.nq / a.pack, a.n_qblocks), dim3(Cfg::THREADS), Cfg::SMEM, s,
                   pages, q, a);
}

// q [n_tokens, nq, D] bfloat16, pages [n_pages, nkv, 4, record]; the rest as gb_attn_prefill_tc.
GB_EXPORT int gb_attn_prefill_kv4(const void* q, const void* pages, const AttnTcArgs* a, float* lse, int n_tokens,
                                  int n_pages, int n_slots, int D, int rows_per_block, cudaStream_t s) {
  if (!q || !pages || !a->out || !a->error || !a->block_table || !a->cu_q || !a->slots || !a->kv_len || a->n_seqs <= 0 ||
      a->nq <= 0 || a->nkv <= 0 || a->nq % a->nkv || a->max_pages <= 0 || a->n_qblocks < 0 || n_tokens <= 0 || n_pages <= 0 ||
      a->chunk < 0 || a->window < 0 || a->keep_first < 0)
    return GB_ERR_BAD_ARG;
  if (a->pack < 1 || a->pack > 64 || (a->pack & (a->pack - 1)) || (a->nq / a->nkv) % a->pack) return GB_ERR_BAD_ARG;
  if ((D != 64 && D != 128) || a->n_qblocks > 65535) return GB_ERR_UNSUPPORTED;
  if (rows_per_block != AT_BM && rows_per_block != 2 * AT_BM) return GB_ERR_BAD_ARG;
  if (((uintptr_t)q | (uintptr_t)pages) & 15) return GB_ERR_BAD_ARG;
  if (a->n_qblocks == 0) return 0;
  const Kv4Pages::Params params = {(const uint8_t*)pages, lse, n_pages, n_slots};
  if (rows_per_block == AT_BM)
    return D == 64 ? launch<1, 1>(params, (const bf16*)q, *a, s) : launch<2, 1>(params, (const bf16*)q, *a, s);
  return D == 64 ? launch<1, 2>(params, (const bf16*)q, *a, s) : launch<2, 2>(params, (const bf16*)q, *a, s);
}
