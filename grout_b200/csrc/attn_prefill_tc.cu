// Prompt attention over pages in bfloat16: the kernel of attn_prefill_tc.cuh with key tiles that TMA brings.
#include "attn_prefill_tc.cuh"

struct TmaPages {
  struct Params {
    CUtensorMap k, v;      // [n_pages * nkv * 64, D] in boxes of 64 rows x 64 elements
  };
  template <int DS, int G>
  using Config = AtConfig<DS, G>;
  __device__ __forceinline__ static constexpr int FULL_ARRIVALS(int) { return 1; }
  __device__ __forceinline__ static constexpr float* lse(const Params&) { return nullptr; }
  __device__ __forceinline__ static int slot(const Params&, int s) { return s; }
  __device__ __forceinline__ static void before_padding() {}
  __device__ __forceinline__ static void cap_scores(float (&s)[AT_BN], const ScoreCap& cap) {
#pragma unroll
    for (int c = 0; c < AT_BN; ++c) s[c] = capped_log2(s[c] * cap.cap_inv, cap);
  }
  __device__ __forceinline__ static void prepare(const Params& p) {
    tma_prefetch_map(&p.k);
    tma_prefetch_map(&p.v);
  }
  // One lane asks for the tiles of the block's list, as stages of the ring come free.
  template <int DS, int G>
  __device__ __forceinline__ static void produce(const Params& p, const AttnTcArgs& a, const AtTiles& b, int) {
    using Cfg = Config<DS, G>;
    constexpr int AT_STAGES = Cfg::STAGES;
    if ((threadIdx.x & 31) == 0) {
      for (int j = 0; j < b.n_tiles; ++j) {
        const int s = j % AT_STAGES;
        // the tile that held this stage has been read by the query blocks that needed it
        const uint32_t par = (((uint32_t)(j / AT_STAGES)) & 1) ^ 1;
        bool freed = j - AT_STAGES >= b.n_a || mbar_wait_idle(&b.kv_empty[s], par, b.abort_flag);
        freed = freed && (j - AT_STAGES >= b.n_b || mbar_wait_idle(&b.kv_empty[AT_STAGES + s], par, b.abort_flag));
        if (!freed) {
          if (!*b.abort_flag) atomicCAS(a.error, 0, GB_ERR_AT_TIMEOUT);
          *b.abort_flag = 1;
          break;
        }
        const int page = b.table[b.tile(j)];
        const int row0 = (page * a.nkv + b.kvh) * AT_BN;
        uint8_t* st = b.kv_s + (size_t)s * Cfg::KV_BYTES;
        mbar_expect_tx(&b.kv_full[s], Cfg::KV_BYTES);
        for (int ds = 0; ds < DS; ++ds) {
          tma_load_2d(st + ds * Cfg::SUB_BYTES, &p.k, ds * 64, row0, &b.kv_full[s]);
          tma_load_2d(st + (DS + ds) * Cfg::SUB_BYTES, &p.v, ds * 64, row0, &b.kv_full[s]);
        }
      }
      pdl_launch_dependents();
    }
  }
};

template <int DS, int G>
static int launch(const TmaPages::Params& pages, const bf16* q, const AttnTcArgs& a, cudaStream_t s) {
  static bool configured = false;
  if (!configured) {
    cudaError_t e = cudaFuncSetAttribute(attn_prefill_tc_kernel<DS, G, TmaPages>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)AtConfig<DS, G>::SMEM);
    if (e != cudaSuccess) return (int)e;
    configured = true;
  }
  return gb_launch(attn_prefill_tc_kernel<DS, G, TmaPages>, dim3(a.nq / a.pack, a.n_qblocks), dim3(AtConfig<DS, G>::THREADS),
                   AtConfig<DS, G>::SMEM, s, pages, q, a);
}

// q [n_tokens, nq, D]; k_pages and v_pages [n_pages, nkv, 64, D]; bf16.
// head_dim 64 or 128 and pages of 64 tokens; anything else is refused
// (GB_ERR_UNSUPPORTED) and the caller uses another kernel.
// rows_per_block 128 or 256 query rows (tokens x a->pack heads); a->n_qblocks counts blocks of that many.
GB_EXPORT int gb_attn_prefill_tc(const void* q, const void* k_pages, const void* v_pages,
                                 const AttnTcArgs* a, int n_tokens, long long n_pages, int D, int page,
                                 int rows_per_block, cudaStream_t s) {
  if (a->chunk < 0) return GB_ERR_BAD_ARG;
  if (!q || !k_pages || !v_pages || !a->out || !a->error || a->n_seqs <= 0 || a->nq <= 0 ||
      a->nkv <= 0 || a->nq % a->nkv || a->max_pages <= 0 || a->n_qblocks < 0 || n_tokens <= 0 ||
      n_pages <= 0)
    return GB_ERR_BAD_ARG;
  if (a->pack < 1 || a->pack > 64 || (a->pack & (a->pack - 1)) || (a->nq / a->nkv) % a->pack) return GB_ERR_BAD_ARG;
  if (page != AT_BN || (D != 64 && D != 128) || a->n_qblocks > 65535) return GB_ERR_UNSUPPORTED;
  if (rows_per_block != AT_BM && rows_per_block != 2 * AT_BM) return GB_ERR_BAD_ARG;
  if (n_pages * a->nkv * AT_BN > 0x7fffffffll) return GB_ERR_UNSUPPORTED;
  if (((uintptr_t)q & 15) != 0) return GB_ERR_BAD_ARG;   // query rows are read 16 bytes at a time
  if (a->n_qblocks == 0) return 0;
  TmaPages::Params pages;
  const uint64_t kv_rows = (uint64_t)n_pages * a->nkv * AT_BN;
  int e = tc_make_map_2d(&pages.k, k_pages, kv_rows, (uint64_t)D, (uint64_t)D * 2, AT_BN, 64);
  if (e) return e;
  e = tc_make_map_2d(&pages.v, v_pages, kv_rows, (uint64_t)D, (uint64_t)D * 2, AT_BN, 64);
  if (e) return e;
  if (rows_per_block == AT_BM)
    return D == 64 ? launch<1, 1>(pages, (const bf16*)q, *a, s) : launch<2, 1>(pages, (const bf16*)q, *a, s);
  return D == 64 ? launch<1, 2>(pages, (const bf16*)q, *a, s) : launch<2, 2>(pages, (const bf16*)q, *a, s);
}
