// The rank numbers of low-rank adapters on the tensor cores: x[t] A_a^T times the adapter's scale, for
// hundreds of tokens and several adapters (adapter.cu has the whole operator).
//
// A tile is 128 tokens (the instruction's rows, one tensor-memory lane each) by the ranks of one adapter
// (its columns, 64 a turn) over a share of K; the shares are the CTAs of a cluster, which leave their sums in
// shared memory and read each other's in rank order. x and A come by TMA. Tokens of other adapters are
// multiplied too and dropped at the end: a tile of prompts has one or two adapters, and x is what the
// kernel reads most of.
//
// What bounds it: the start and the end of a CTA (barriers, tensor memory, the meeting of the shares) around
// a stream of (128 + ranks) * 128 bytes a K block. 2,048 tokens of 4,096 at rank 48, one or two adapters a
// block: 9.9 us in graph replays, where x and A alone are 18 MB, 2.7 us at the copy rate. (With mma.sync
// instead, from registers or through cp.async stages, the same took 15 to 40 us: the instructions' own rate.)
#define FB_STATUS_KERNEL 6
#include "adapter_planes.cuh"
#include "gemm_tcgen05.cuh"

namespace {

constexpr int BLOCK_ROWS = 256;  // tokens of a block of planes: a tile of the paired product
constexpr int MAX_SLOTS = 1024;

template <int RB>
struct LowSmem {
  static constexpr int X_BYTES = BM * BK * 2;
  static constexpr int STAGE_BYTES = X_BYTES + RB * BK * 2;
  static constexpr int PART_BYTES = BM * (RB + 1) * 4;  // this CTA's share of K
  // two CTAs an SM: the start and the end of one beside the stream of the other
  static constexpr int STAGES = RB <= 32 ? 4 : 3;
  static constexpr int BYTES = STAGES * STAGE_BYTES + 1024 /*align*/ + PART_BYTES + 256;
};

__device__ __forceinline__ void cluster_barrier() {
  __syncwarp();  // the aligned form wants whole warps
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_peer(const float* mine, unsigned rank) {
  uint32_t remote;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(mine)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
  return v;
}

// CTA (i, y, z): 128 tokens, the adapters y, y + gridDim.y, .. of their block, share z of K. PLANES: a block
// is 256 tokens, and every adapter of it gets a plane of rows (adapter_planes.cuh), zero in those of others; else a
// block is the tile, and a token's own rank numbers go to its row of `low`.
template <int RB, bool PLANES>
__global__ void __launch_bounds__(THREADS, 2)
adapter_low_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_a,
                   const float* scales, const int* index, int slots, int rank, int T, int K, int most,
                   __nv_bfloat16* u, int* counts, int* slots_of, float* low) {
  using S = LowSmem<RB>;
  constexpr int TMEM_COLS = RB < 32 ? 32 : RB;
  constexpr int ROWS = PLANES ? BLOCK_ROWS : BM;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* tiles = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  float (*part)[RB + 1] = (float (*)[RB + 1])(tiles + S::STAGES * S::STAGE_BYTES);
  uint64_t* full = (uint64_t*)((uint8_t*)part + S::PART_BYTES);
  uint64_t* empty = full + S::STAGES;
  uint64_t* acc_full = empty + S::STAGES;
  uint32_t* tmem_slot = (uint32_t*)(acc_full + 1);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
  __shared__ unsigned s_present[MAX_SLOTS / 32], s_before[MAX_SLOTS / 32];
  __shared__ int s_index[BM], s_listed[BLOCK_ROWS], s_count;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int t0 = blockIdx.x * BM, block = t0 / ROWS;
  const int shares = gridDim.z, share = blockIdx.z;
  if (tid == 0) {
    for (int s = 0; s < S::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (tid < MAX_SLOTS / 32) s_present[tid] = 0u;
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"((uint32_t)TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // the adapters of the block, by their slots
  fb_pdl_wait();
  int slot_of[(ROWS + THREADS - 1) / THREADS];
#pragma unroll
  for (int i = 0; i < (ROWS + THREADS - 1) / THREADS; ++i) {
    const int r = tid + i * THREADS, t = block * ROWS + r;
    int slot = r < ROWS && t < T ? index[t] : -1;
    if (slot >= slots || slot < 0) slot = -1;
    else atomicOr(&s_present[slot >> 5], 1u << (slot & 31));
    slot_of[i] = slot;
    if (r < ROWS && t >= t0 && t < t0 + BM) s_index[t - t0] = slot;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  if (warp == 0) {  // how many stand in front of each word's
    const unsigned word = s_present[lane];
    unsigned upto = __popc(word);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned other = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += other;
    }
    if (lane == 31) s_count = (int)upto;
    s_before[lane] = upto - __popc(word);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < (ROWS + THREADS - 1) / THREADS; ++i) {
    const int slot = slot_of[i];
    if (slot >= 0)  // (several threads may say the same)
      s_listed[s_before[slot >> 5] + __popc(s_present[slot >> 5] & ((1u << (slot & 31)) - 1))] = slot;
  }
  __syncthreads();
  const int count = s_count;
  if constexpr (PLANES) {
    if (t0 % BLOCK_ROWS == 0 && share == 0 && blockIdx.y == 0) {
      if (tid == 0) counts[block] = count;
      for (int i = tid; i < count; i += THREADS) slots_of[block * most + i] = s_listed[i];
    }
  }

  const int nkb = (K + BK - 1) / BK, each = (nkb + shares - 1) / shares;
  const int kb0 = min(nkb, share * each), n = min(nkb, kb0 + each) - kb0;  // this share's K blocks
  int it = 0, turn = 0;
  for (int e = blockIdx.y; e < count; e += gridDim.y) {
    const int slot = s_listed[e];
    const int width = fb_plane_width(rank);
    __nv_bfloat16* rows = PLANES ? u + ((size_t)(block * most + e) * BLOCK_ROWS + t0 % BLOCK_ROWS) * width : nullptr;
    if (!__syncthreads_or(tid < BM && s_index[tid & (BM - 1)] == slot)) {  // none of these tokens: zeros
      if (PLANES && share == 0) {
        const int live = min(BM, T - t0);
        for (int i = tid; i < live * width / 8; i += THREADS)
          reinterpret_cast<uint4*>(rows)[i] = make_uint4(0u, 0u, 0u, 0u);
      }
      continue;
    }
    const float scale = scales[slot];
    for (int r0 = 0; r0 < rank; r0 += RB, it += n, ++turn) {
      if (warp == 0) {
        if (lane == 0) {  // TMA producer
          for (int i = 0; i < n; ++i) {
            const int use = it + i, s = use % S::STAGES;
            if (!mbar_wait(&empty[s], ((uint32_t)(use / S::STAGES) & 1u) ^ 1u, abort_flag, 1, i)) break;
            uint8_t* x_dst = tiles + s * S::STAGE_BYTES;
            mbar_expect_tx(&full[s], S::STAGE_BYTES);
            tma_load_2d(x_dst, &map_x, &full[s], (kb0 + i) * BK, t0);
            tma_load_2d(x_dst + S::X_BYTES, &map_a, &full[s], (kb0 + i) * BK, slot * rank + r0);
          }
        }
      } else if (warp == 1) {
        if (lane == 0) {  // MMA issuer
          constexpr uint32_t idesc = make_idesc(BM, RB);
          bool ok = true;
          for (int i = 0; i < n && ok; ++i) {
            const int use = it + i, s = use % S::STAGES;
            ok = mbar_wait(&full[s], (uint32_t)(use / S::STAGES) & 1u, abort_flag, 2, i);
            if (!ok) break;
            tc_fence_after();
            const uint32_t x_addr = smem_u32(tiles + s * S::STAGE_BYTES), a_addr = x_addr + S::X_BYTES;
#pragma unroll
            for (int k = 0; k < BK / UMMA_K; ++k)
              umma(tmem_base, make_desc(x_addr + k * UMMA_K * 2), make_desc(a_addr + k * UMMA_K * 2), idesc,
                   (i | k) != 0 ? 1u : 0u);
            tc_commit(&empty[s]);
          }
          if (ok && n > 0) tc_commit(acc_full);
        }
      } else {
        const int quarter = warp & 3, t = quarter * 32 + lane;  // the TMEM lanes this warp may read
        const bool ok = __all_sync(0xffffffffu, n > 0 && mbar_wait(acc_full, (uint32_t)turn & 1u, abort_flag, 3, turn));
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < RB; c += 16) {
          uint32_t v[16];
          if (ok) {
            tmem_ld16(tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)c, v);
            tmem_ld_wait();
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) part[t][c + j] = ok ? __uint_as_float(v[j]) : 0.f;
        }
        tc_fence_before();
      }
      __syncthreads();
      if (shares > 1) cluster_barrier();
      tc_fence_after();
      // the cluster's CTAs share the tokens; a token's ranks side by side
      const int wide = min(RB, rank - r0), mine = BM / shares;
      const int reach = PLANES ? fb_plane_ranks(wide) : wide;  // (a plane's ranks behind the last one are zeros)
      for (int i = tid; i < mine * reach; i += THREADS) {
        const int t = share * mine + i / reach, j = i % reach;
        if (t0 + t >= T) break;
        const bool own = s_index[t] == slot;
        float v = 0.f;
        if (PLANES && (j >= wide || !own)) {
        } else if (shares > 1) {
          float p[8];
#pragma unroll
          for (int z = 0; z < 8; ++z) p[z] = z < shares ? ld_peer(&part[t][j], z) : 0.f;
#pragma unroll
          for (int z = 0; z < 8; ++z) v += p[z];
        } else {
          v = part[t][j];
        }
        if constexpr (PLANES) fb_store_halves(rows + (size_t)t * width, r0 + j, own && j < wide ? scale * v : 0.f);
        else if (own) low[(size_t)(t0 + t) * rank + r0 + j] = scale * v;
      }
      // nobody's sums are overwritten, or gone, while a peer still reads them
      if (shares > 1) cluster_barrier(); else __syncthreads();
    }
  }
  // ------------------------------------------------------------------ teardown
  if (tid == 0 && *abort_flag) {  // after a wait that ran out: what is still on its way lands first
    for (int s = 0; s < S::STAGES; ++s)
      for (uint32_t spin = 0; spin < (SPIN_LIMIT >> 4) && !mbar_try_wait(&full[s], (uint32_t)(it / S::STAGES) & 1u); ++spin) {}
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                 "r"((uint32_t)TMEM_COLS)
                 : "memory");
  }
}

template <int RB, bool PLANES>
int launch_low(const CUtensorMap& mx, const CUtensorMap& ma, const float* scales, const int* index, int slots,
               int rank, int T, int K, int most, int side, int shares, __nv_bfloat16* u, int* counts,
               int* slots_of, float* low, cudaStream_t stream) {
  static bool seen[64] = {};
  if (fb_first_use_on_device(seen)) {
    cudaError_t e = cudaFuncSetAttribute(adapter_low_kernel<RB, PLANES>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, LowSmem<RB>::BYTES);
    if (e != cudaSuccess) return fb_fail(2, "adapter_low: shared memory opt-in: %s", cudaGetErrorString(e));
  }
  fb_launch_cluster(adapter_low_kernel<RB, PLANES>, dim3((T + BM - 1) / BM, side, shares), dim3(THREADS),
                    LowSmem<RB>::BYTES, stream, (unsigned)shares, mx, ma, scales, index, slots, rank, T, K, most,
                    u, counts, slots_of, low);
  return fb_check_launch("adapter_low");
}
}  // namespace

// u != null: planes for fb_gemm_tc_adapted, u [ceil(T / 256) * most * 256, fb_plane_width(rank)] bfloat16, counts [blocks],
// slots_of [blocks, most]; rows behind the last token are left as they are (what the product makes of them
// goes nowhere). Else: low [T, rank] float32, rows of tokens without an adapter left as they are. `most`: at
// least the adapters that one block (256 tokens, or 128) can have. side: CTAs that share the adapters of a
// block; shares: CTAs that split K (1, 2, 4 or 8).
FB_API int fb_adapter_low(const void* x, long long ldx, const void* a, const float* scales, const int* index,
                          int slots, int rank, int T, int K, int most, int side, int shares, void* u,
                          int* counts, int* slots_of, float* low, cudaStream_t stream) {
  FB_REQUIRE(T > 0 && K > 0 && rank > 0 && rank % 8 == 0 && slots > 0 && slots <= MAX_SLOTS && ldx >= K,
             "adapter_low: bad sizes T=%d K=%d rank=%d slots=%d", T, K, rank, slots);
  const int of_block = u != nullptr ? BLOCK_ROWS : BM;
  FB_REQUIRE(most >= (slots < of_block ? slots : of_block) || most >= T, "adapter_low: room for %d adapters a block", most);
  FB_REQUIRE(K % 8 == 0 && ldx % 8 == 0 && (((uintptr_t)x | (uintptr_t)a | (uintptr_t)u) % 16) == 0,
             "adapter_low: K, the row stride and the operands must keep 16-byte alignment");
  FB_REQUIRE((shares == 1 || shares == 2 || shares == 4 || shares == 8) && side > 0 && side <= 256,
             "adapter_low: %d shares of K, %d of the adapters", shares, side);
  FB_REQUIRE(u != nullptr ? counts != nullptr && slots_of != nullptr : low != nullptr, "adapter_low: no place for the results");
  bind_status_mirror(stream);
  const int rb = rank <= 16 ? 16 : rank <= 32 ? 32 : 64;
  CUtensorMap mx, ma;
  int rc = make_map(&mx, x, T, K, ldx, BM);
  if (!rc) rc = make_map(&ma, a, (long long)slots * rank, K, K, rb);
  if (rc) return rc;
#define FB_LOW(RB, PLANES)                                                                                   \
  return launch_low<RB, PLANES>(mx, ma, scales, index, slots, rank, T, K, most, side, shares,                 \
                                (__nv_bfloat16*)u, counts, slots_of, low, stream)
  if (u != nullptr) {
    if (rb == 16) FB_LOW(16, true);
    if (rb == 32) FB_LOW(32, true);
    FB_LOW(64, true);
  }
  if (rb == 16) FB_LOW(16, false);
  if (rb == 32) FB_LOW(32, false);
  FB_LOW(64, false);
#undef FB_LOW
}

// As fb_gemm_tc_status, for the kernels of this file.
FB_API int fb_adapter_status(int* detail) {
  int host[4] = {0, 0, 0, 0};
  cudaError_t e = cudaMemcpyFromSymbol(host, g_status, sizeof(host));
  if (e != cudaSuccess) return fb_fail(2, "adapter_status: %s", cudaGetErrorString(e));
  if (detail) { detail[0] = host[1]; detail[1] = host[2]; detail[2] = host[3]; }
  if (host[0]) {
    int zero[4] = {0, 0, 0, 0};
    cudaMemcpyToSymbol(g_status, zero, sizeof(zero));
  }
  return host[0] ? host[1] : 0;
}
