// Low-rank adapters of many requests beside a shared projection:
//     out[r] = y[r] + scale[a] * (x[r] . down[a]^T) . up[a]^T,   a = the adapter of row r
// A packed projection has a `down` of its own for each part; a column of `up` meets the inner values of its part.
//
// The plan (one block, once per step) sorts the rows by adapter into tiles of at most `tile_rows` rows of one adapter.  A product is then
// one launch: a cluster of blocks takes a tile.  Its blocks share the input channels, so that a tile's `down` is fetched by many
// multiprocessors at once; their partial inner values are summed through distributed shared memory, in a fixed order; then the blocks
// share the output columns.  `up` comes into shared memory meanwhile, as far as there is room.
//
// Precision: bf16 operands, 32-bit sums.  The inner values are scaled in 32 bits and enter the second product as two bf16 terms (16 bits of
// mantissa): rounded to one they would cost the sum as much as its own rounding does.
#include "dec_common.cuh"

namespace b200kv {

constexpr int kAdThreads = 256;
constexpr int kAdWarps = kAdThreads / 32;
constexpr int kAdMaxParts = 4;
constexpr int kAdMaxSlots = 4096;
constexpr int kAdPlanThreads = 1024;
constexpr int kAdSimtChannels = 512;  // input channels that the CUDA cores' form stages at a time
constexpr int kAdMaxInner = 192;      // inner values of a row in tiles of 64 rows
constexpr int kAdChannels = 64;       // input channels of a stage there

struct AdArgs {
  const void *down, *up;
  const float* scale;
  const void *x, *y;
  void* out;
  long long x_stride, y_stride, out_stride;
  const int32_t* order;
  const int4* tiles;
  int tile_rows;  // of the plan
  int rank, width, parts;
  int ends[kAdMaxParts];
  int groups;           // of 32 output columns, none across parts
  int inner;            // parts * rank
  int inner_row;        // floats between rows of partial inner values
  int t_row;            // bytes between rows of finished ones
  int u_row;            // bytes between columns of `up` in shared memory
  int vec;              // y and out rows can be read and written in 16 bytes
  uint32_t off_t, off_u;  // shared memory: the finished inner values, `up`
};

// ---------------------------------------------------------------------------------------------------------------- the plan
// Tile i has rows order[i * tile_rows ..], -1 behind them.  Which rows of one adapter are where is left to atomics: a row's result does not
// depend on its place.
__global__ void __launch_bounds__(kAdPlanThreads)
adapter_plan_kernel(const int32_t* ids, int N, int slots, int tile_rows, int32_t* order, int4* tiles, int max_tiles, int32_t* status) {
  extern __shared__ int ad_plan_smem[];  // rows of each group, then where its next row goes; group `slots`: no adapter
  __shared__ int warp_tiles[32];
  pdl_enter();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x;
  for (int g = tid; g <= slots; g += threads) ad_plan_smem[g] = 0;
  for (int i = tid; i < max_tiles * tile_rows; i += threads) order[i] = -1;
  __syncthreads();
  auto group = [&](int r) {
    const int id = ids[r];
    if (id >= 0 && id < slots) return id;
    if (id != -1 && status) atomicOr(status, B200KV_S_BAD_POSITION);
    return slots;
  };
  for (int base = warp * 32; base < N; base += threads) {
    const int r = base + lane;
    const unsigned on = __ballot_sync(0xffffffffu, r < N);
    if (r < N) {
      const int g = group(r);
      const unsigned same = __match_any_sync(on, g);
      if (lane == __ffs(same) - 1) atomicAdd(&ad_plan_smem[g], __popc(same));
    }
  }
  __syncthreads();
  int tiles_before = 0;
  for (int base = 0; base <= slots; base += threads) {
    const int g = base + tid, n = g <= slots ? ad_plan_smem[g] : 0, t = (n + tile_rows - 1) / tile_rows;
    int ts = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int b = __shfl_up_sync(0xffffffffu, ts, o);
      if (lane >= o) ts += b;
    }
    if (lane == 31) warp_tiles[warp] = ts;
    __syncthreads();
    int tw = tiles_before, ta = 0;
    for (int w = 0; w < threads / 32; ++w) {
      if (w < warp) tw += warp_tiles[w];
      ta += warp_tiles[w];
    }
    const int tile = tw + ts - t;
    if (g <= slots) {
      ad_plan_smem[g] = tile * tile_rows;
      for (int i = 0; i < t; ++i)
        if (tile + i < max_tiles) tiles[tile + i] = make_int4(g < slots ? g : -1, min(tile_rows, n - i * tile_rows), 0, 0);
    }
    tiles_before += ta;
    __syncthreads();
  }
  for (int i = tiles_before + tid; i < max_tiles; i += threads) tiles[i] = make_int4(-1, 0, 0, 0);
  for (int base = warp * 32; base < N; base += threads) {
    const int r = base + lane;
    const unsigned on = __ballot_sync(0xffffffffu, r < N);
    if (r < N) {
      const int id = ids[r], g = id >= 0 && id < slots ? id : slots;
      const unsigned same = __match_any_sync(on, g);
      int at = 0;
      if (lane == __ffs(same) - 1) at = atomicAdd(&ad_plan_smem[g], __popc(same));
      at = __shfl_sync(same, at, __ffs(same) - 1);
      order[at + __popc(same & ((1u << lane) - 1))] = r;
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------- shared pieces
__device__ __forceinline__ void ad_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t ad_cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void ad_cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void ad_cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ uint32_t ad_at_rank(uint32_t local, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  return remote;
}
__device__ __forceinline__ float4 ad_ld_remote4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void ad_st_remote2(uint32_t addr, uint32_t a, uint32_t b) {
  asm volatile("st.shared::cluster.v2.b32 [%0], {%1,%2};" ::"r"(addr), "r"(a), "r"(b) : "memory");
}
__device__ __forceinline__ void ad_copy16(uint32_t dst, const void* src, int bytes) {  // zeros behind the first `bytes`
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void ad_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void ad_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(kLeft) : "memory"); }

// Column group g (of 32): its part, first column and the end of its part's columns.
struct AdGroup { int part, col, end; };
__device__ __forceinline__ AdGroup ad_group(const AdArgs& a, int g) {
  int begin = 0;
#pragma unroll
  for (int p = 0; p < kAdMaxParts; ++p) {
    if (p < a.parts) {
      const int n = (a.ends[p] - begin + 31) >> 5;
      if (g < n) return {p, begin + 32 * g, a.ends[p]};
      g -= n;
      begin = a.ends[p];
    }
  }
  return {0, 0, 0};
}
template <int kC>
__device__ __forceinline__ int ad_first_group(const AdArgs& a, int rank) { return (int)((unsigned)a.groups * (unsigned)rank / kC); }

// Rows of the tile without an adapter: copied where the result has a place of its own.
template <typename T, int kC>
__device__ __forceinline__ void ad_copy_rows(const AdArgs& a, const int32_t* order, int count, int rank) {
  if (a.out == a.y) return;
  const int lo = ad_first_group<kC>(a, rank), hi = ad_first_group<kC>(a, rank + 1);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int g = lo + warp; g < hi; g += kAdWarps) {
    const AdGroup gr = ad_group(a, g);
    if (gr.col + lane >= gr.end) continue;
    for (int i = 0; i < count; ++i) {
      const long long r = order[i];
      ((T*)a.out)[r * a.out_stride + gr.col + lane] = ((const T*)a.y)[r * a.y_stride + gr.col + lane];
    }
  }
}

// Four finished inner values as two bf16 terms each.
__device__ __forceinline__ void ad_split(const float4& s, uint2& hi, uint2& lo) {
  const float f[4] = {s.x, s.y, s.z, s.w};
  uint32_t h[4], l[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    h[j] = float_to_bf16_bits(f[j]);
    const float rest = f[j] - bf16_bits_to_float(h[j]);
    l[j] = fabsf(rest) < INFINITY ? float_to_bf16_bits(rest) : 0u;  // (an infinite or NaN value has no second term)
  }
  hi = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
  lo = make_uint2(l[0] | (l[1] << 16), l[2] | (l[3] << 16));
}

// Sum over the cluster's blocks of the partial values at an offset of shared memory.
template <int kC>
__device__ __forceinline__ float4 ad_total(uint32_t at, float scale) {
  float4 v[kC];
#pragma unroll
  for (int q = 0; q < kC; ++q) v[q] = ad_ld_remote4(ad_at_rank(at, q));
  float4 s = v[0];
#pragma unroll
  for (int q = 1; q < kC; ++q) { s.x += v[q].x; s.y += v[q].y; s.z += v[q].z; s.w += v[q].w; }
  s.x *= scale; s.y *= scale; s.z *= scale; s.w *= scale;
  return s;
}

// ---------------------------------------------------------------------------------------------------------------- tensor cores
// kRows 16: the warps share the block's channels and, where there are more than 64 inner values, those too; both operands go straight
// from memory to registers.  kRows 64: a warp takes sixteen rows and half the channels, `down` is staged in shared memory for all of them.
// kNT: blocks of eight inner values of a warp.  kKB: blocks of sixteen inner values of a part.  kC: blocks of a cluster.  kStages: chunks of columns of
// `up` that are in shared memory or on their way.
// The order of a product's channels is free, so that a lane loads whole 16 bytes: lane t of a row's four has channels 8t .. 8t + 7 of 32.
template <int kRows, int kNT, int kKB, int kC, int kStages>
__global__ void __launch_bounds__(kAdThreads, kKB > 4 ? 1 : (kRows == 16 ? 3 : 2)) adapter_kernel(const __grid_constant__ AdArgs a) {
  extern __shared__ __align__(16) uint8_t ad_smem[];
  constexpr int kGroups = kRows == 16 ? 8 : 4;     // column groups of a chunk
  constexpr int kM = kRows == 16 ? 1 : 2;          // blocks of sixteen rows that a warp adds up in the second product
  const uint32_t smem = (uint32_t)__cvta_generic_to_shared(ad_smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, t = lane & 3;
  const int rank = (int)ad_cluster_rank(), cl = blockIdx.x / kC;
  pdl_enter();
  pdl_wait();
  const int subs = a.tile_rows / kRows;
  const int4 tile = a.tiles[cl / subs];
  const int32_t* order = a.order + (long long)cl * kRows;
  const int slot = tile.x, count = min(tile.y - (cl % subs) * kRows, kRows);
  const int m0 = kRows == 16 ? 0 : 16 * (warp & 3);
  const int row0 = order[m0 + gid], row1 = order[m0 + gid + 8];
  if (count <= 0) return;  // (with the whole cluster)
  if (slot < 0) return ad_copy_rows<uint16_t, kC>(a, order, count, rank);
  const uint16_t* down = (const uint16_t*)a.down + (long long)slot * a.inner * a.width;
  const uint16_t* up = (const uint16_t*)a.up + (long long)slot * a.ends[a.parts - 1] * a.rank;
  const uint4 zero4 = make_uint4(0, 0, 0, 0);
  const int chunks = (a.width + 31) >> 5;
  float* part = reinterpret_cast<float*>(ad_smem);
  const int g0 = ad_first_group<kC>(a, rank), g1 = ad_first_group<kC>(a, rank + 1);

  // This warp's group of each chunk, and where its columns of `up` go.  Column 8 (n / 2) + 2 j + n % 2 of a group lies at 8 j + n: see below.  In tiles of 64
  // rows two warps share a group, and each brings half of it.
  const int mine = kRows == 16 ? warp : warp & 3, rows_at = kRows == 16 ? 0 : 32 * (warp >> 2);
  const uint32_t u_at = a.off_u + mine * 32 * a.u_row;
  const int u_stage = kGroups * 32 * a.u_row, vecs = a.rank >> 3;
  const unsigned by_vecs = (65536u + vecs - 1) / vecs;  // i / vecs of i < 512 by a product
  auto fetch_up = [&](const AdGroup& gr, int stage) {
    const uint16_t* src = up + (long long)gr.col * a.rank;
    const uint32_t dst = smem + u_at + stage * u_stage;
    const int n = gr.end ? 32 * vecs : 0;  // (a stage behind the last group may have no place)
    for (int i = kRows == 16 ? lane : lane + (warp & 4) * 8; i < n; i += kRows == 16 ? 32 : 64) {
      const int c = (int)((unsigned)i * by_vecs >> 16), v = i - c * vecs;
      const int place = 8 * ((c >> 1) & 3) + 2 * (c >> 3) + (c & 1);
      const bool in = gr.col + c < gr.end;
      ad_copy16(dst + place * a.u_row + v * 16, in ? src + i * 8 : up, in ? 16 : 0);
    }
    ad_commit();
  };
  AdGroup ring[kStages];  // the groups in the stages
#pragma unroll
  for (int i = 0; i < kStages; ++i) ring[i] = g0 + mine + i * kGroups < g1 ? ad_group(a, g0 + mine + i * kGroups) : AdGroup{0, 0, 0};
  auto fetch_first = [&]() {
#pragma unroll
    for (int i = 0; i < kStages; ++i) fetch_up(ring[i], i);
  };

  float acc[kNT][4];
#pragma unroll
  for (int n = 0; n < kNT; ++n)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[n][j] = 0.f;
  const uint16_t* x0 = (const uint16_t*)a.x + (long long)max(row0, 0) * a.x_stride;
  const uint16_t* x1 = (const uint16_t*)a.x + (long long)max(row1, 0) * a.x_stride;
  auto load_x = [&](const uint16_t* x, int row, int k) { return row >= 0 && k < a.width ? *reinterpret_cast<const uint4*>(x + k) : zero4; };

  if constexpr (kRows == 16) {
    const int wn = (a.inner + 8 * kNT - 1) / (8 * kNT);                // warps side by side over the inner values
    const int across = wn <= 1 ? 1 : (wn <= 2 ? 2 : (wn <= 4 ? 4 : 8)), deep = kAdWarps / across;
    const int n0 = (warp % across) * kNT * 8, d = warp / across;
    bool first = true;
    for (int c = rank * deep + d; c < chunks || first; c += kC * deep) {
      const int k = 32 * c + 8 * t;  // (the width is a multiple of 8)
      uint4 w[kNT];
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        const int j = n0 + 8 * n + gid;
        w[n] = k < a.width && j < a.inner ? __ldg(reinterpret_cast<const uint4*>(down + (long long)j * a.width + k)) : zero4;
      }
      const uint4 u0 = load_x(x0, row0, k), u1 = load_x(x1, row1, k);
      if (first) {
        fetch_first();
        first = false;
      }
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        ad_mma(acc[n], u0.x, u1.x, u0.y, u1.y, w[n].x, w[n].y);
        ad_mma(acc[n], u0.z, u1.z, u0.w, u1.w, w[n].z, w[n].w);
      }
    }
    // the warps' shares of the channels, in order: [deep][16][inner_row]
    float* mine = part + d * 16 * a.inner_row;
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
      const int j = n0 + 8 * n + 2 * t;
      if (j < a.inner) {
        *reinterpret_cast<float2*>(mine + gid * a.inner_row + j) = make_float2(acc[n][0], acc[n][1]);
        *reinterpret_cast<float2*>(mine + (gid + 8) * a.inner_row + j) = make_float2(acc[n][2], acc[n][3]);
      }
    }
    __syncthreads();
    const int quads = a.inner >> 2;
    for (int i = tid; i < count * quads; i += kAdThreads) {
      const int row = i / quads, at = row * a.inner_row + (i - row * quads) * 4;
      float4 s = *reinterpret_cast<const float4*>(part + at);
      for (int q = 1; q < deep; ++q) {
        const float4 v = *reinterpret_cast<const float4*>(part + q * 16 * a.inner_row + at);
        s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
      }
      *reinterpret_cast<float4*>(part + at) = s;
    }
  } else {
    // stages of 64 channels, two in shared memory; the half that a warp takes of each lies 64 bytes apart in odd rows, so that two rows are at
    // different banks
    const int c0 = (int)((long long)((chunks + 1) / 2) * rank / kC), c1 = (int)((long long)((chunks + 1) / 2) * (rank + 1) / kC);
    const int half = warp >> 2, stage_bytes = a.inner * 128;
    auto fetch_down = [&](int c) {
      if (c < c1) {
        const uint32_t stage = smem + (c & 1) * stage_bytes;
        for (int i = tid; i < a.inner * 8; i += kAdThreads) {
          const int j = i >> 3, v = i & 7, k = kAdChannels * c + 8 * v;
          ad_copy16(stage + j * 128 + ((v ^ ((j & 1) << 2)) << 4), down + (k < a.width ? (long long)j * a.width + k : 0), k < a.width ? 16 : 0);
        }
      }
      ad_commit();
    };
    fetch_down(c0);
    uint4 u0 = load_x(x0, row0, kAdChannels * c0 + 32 * half + 8 * t), u1 = load_x(x1, row1, kAdChannels * c0 + 32 * half + 8 * t);
    for (int c = c0; c < c1; ++c) {
      fetch_down(c + 1);
      const int k = kAdChannels * (c + 1) + 32 * half + 8 * t;
      const uint4 v0 = c + 1 < c1 ? load_x(x0, row0, k) : zero4, v1 = c + 1 < c1 ? load_x(x1, row1, k) : zero4;
      ad_wait<1>();
      __syncthreads();
      if (m0 < count) {
        const uint8_t* stage = ad_smem + (c & 1) * stage_bytes + gid * 128 + (((half * 4 + t) ^ ((gid & 1) << 2)) << 4);
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
          if (8 * n < a.inner) {
            const uint4 w = *reinterpret_cast<const uint4*>(stage + n * 1024);
            ad_mma(acc[n], u0.x, u1.x, u0.y, u1.y, w.x, w.y);
            ad_mma(acc[n], u0.z, u1.z, u0.w, u1.w, w.z, w.w);
          }
        }
      }
      u0 = v0;
      u1 = v1;
      __syncthreads();
    }
    ad_wait<0>();
    __syncthreads();
    fetch_first();
    // one half's values, then both
#pragma unroll
    for (int h = 1; h >= 0; --h) {
      if (half == h && m0 < count) {
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
          if (8 * n < a.inner) {
            float2* p0 = reinterpret_cast<float2*>(part + (m0 + gid) * a.inner_row + 8 * n + 2 * t);
            float2* p1 = p0 + 4 * a.inner_row;
            const float2 q0 = h ? make_float2(0.f, 0.f) : *p0, q1 = h ? make_float2(0.f, 0.f) : *p1;
            *p0 = make_float2(acc[n][0] + q0.x, acc[n][1] + q0.y);
            *p1 = make_float2(acc[n][2] + q1.x, acc[n][3] + q1.y);
          }
        }
      }
      if (h) __syncthreads();
    }
  }
  ad_cluster_arrive();

  // ---- the second product: 32 columns of a warp at a time, as four tiles of eight.  Tile j's column n is column 8 (n / 2) + 2 j + n % 2 of the 32, so that a
  // lane has eight columns side by side.  Lane t of a row's four has inner values 4t .. 4t + 3 of sixteen; where eight are left over, the two
  // terms of 2t and 2t + 1 share one step.
  int rows[2 * kM];
#pragma unroll
  for (int i = 0; i < 2 * kM; ++i) rows[i] = order[rows_at + gid + 8 * i];
  const uint16_t* y = (const uint16_t*)a.y;
  uint16_t* out = (uint16_t*)a.out;
  uint4 yv[2 * kM];
  auto load_y = [&](const AdGroup& gr) {
    const int col = gr.col + 8 * t;
    const bool whole = a.vec && gr.end - col >= 8;
#pragma unroll
    for (int i = 0; i < 2 * kM; ++i) yv[i] = rows[i] >= 0 && whole ? *reinterpret_cast<const uint4*>(y + (long long)rows[i] * a.y_stride + col) : zero4;
  };
  load_y(ring[0]);  // (on its way while the inner values are exchanged)

  const int p0 = g0 < g1 ? ad_group(a, g0).part : 0, width_t = g0 < g1 ? (ad_group(a, g1 - 1).part - p0 + 1) * a.rank : 0;
  const float scale = a.scale[slot];
  ad_cluster_wait();
  if constexpr (kRows == 16) {
    // every block takes what its columns need from all of them
    const int quads = width_t >> 2;
    for (int i = tid; i < count * quads; i += kAdThreads) {
      const int row = i / quads, col = (i - row * quads) * 4;
      uint2 hi, lo;
      ad_split(ad_total<kC>(smem + (row * a.inner_row + p0 * a.rank + col) * 4, scale), hi, lo);
      uint8_t* to = ad_smem + a.off_t + row * a.t_row + col * 2;
      *reinterpret_cast<uint2*>(to) = hi;
      *reinterpret_cast<uint2*>(to + width_t * 2) = lo;
    }
    ad_cluster_arrive();  // nobody reads another block's memory behind this
  } else {
    // every block sums a share of the rows over all blocks and hands it to the ones whose columns need it
    const int quads = a.inner >> 2, n = count * quads;
    for (int i = rank * kAdThreads + tid; i < n; i += kC * kAdThreads) {
      const int row = i / quads, col = (i - row * quads) * 4, p = col / a.rank;
      uint2 hi, lo;
      ad_split(ad_total<kC>(smem + (row * a.inner_row + col) * 4, scale), hi, lo);
#pragma unroll
      for (int q = 0; q < kC; ++q) {
        const int q0 = ad_first_group<kC>(a, q), q1 = ad_first_group<kC>(a, q + 1);
        if (q0 >= q1) continue;
        const int first = ad_group(a, q0).part, last = ad_group(a, q1 - 1).part;
        if (p < first || p > last) continue;
        const uint32_t dst = ad_at_rank(smem + a.off_t + row * a.t_row + (col - first * a.rank) * 2, q);
        ad_st_remote2(dst, hi.x, hi.y);
        ad_st_remote2(dst + (last - first + 1) * a.rank * 2, lo.x, lo.y);
      }
    }
    ad_cluster_arrive();
    ad_cluster_wait();
  }

  const int full = a.rank >> 4;
  const bool tail = a.rank & 8;
  if (kRows == 16) __syncthreads();  // the finished inner values
  auto pair_sync = [&]() {  // of the warps that share a group
    if (kRows == 16) __syncwarp();
    else asm volatile("bar.sync %0, 64;" ::"r"(mine + 1) : "memory");
  };
  for (int g = g0 + mine, stage = 0; g < g1; g += kGroups, stage = stage + 1 == kStages ? 0 : stage + 1) {
    ad_wait<kStages - 1>();
    pair_sync();
    {
      const AdGroup now = ring[0];
#pragma unroll
      for (int i = 0; i + 1 < kStages; ++i) ring[i] = ring[i + 1];
      ring[kStages - 1] = g + kStages * kGroups < g1 ? ad_group(a, g + kStages * kGroups) : AdGroup{0, 0, 0};
      uint4 v[2 * kM];
#pragma unroll
      for (int i = 0; i < 2 * kM; ++i) v[i] = yv[i];
      load_y(ring[0]);
      const uint8_t* us = ad_smem + u_at + stage * u_stage + gid * a.u_row;
      const uint8_t* ts = ad_smem + a.off_t + (now.part - p0) * a.rank * 2;
      float d[kM][4][4];
#pragma unroll
      for (int m = 0; m < kM; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) d[m][j][i] = 0.f;
#pragma unroll
      for (int kb = 0; kb < kKB; ++kb) {
        if (kb < full) {
          uint2 b[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) b[j] = *reinterpret_cast<const uint2*>(us + 8 * j * a.u_row + 32 * kb + 8 * t);
#pragma unroll
          for (int m = 0; m < kM; ++m) {
            const uint8_t* t0 = ts + (rows_at + 16 * m + gid) * a.t_row + 32 * kb + 8 * t;
            const uint8_t* t1 = t0 + 8 * a.t_row;
            const uint2 h0 = *reinterpret_cast<const uint2*>(t0), h1 = *reinterpret_cast<const uint2*>(t1);
            const uint2 l0 = *reinterpret_cast<const uint2*>(t0 + width_t * 2), l1 = *reinterpret_cast<const uint2*>(t1 + width_t * 2);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              ad_mma(d[m][j], h0.x, h1.x, h0.y, h1.y, b[j].x, b[j].y);
              ad_mma(d[m][j], l0.x, l1.x, l0.y, l1.y, b[j].x, b[j].y);
            }
          }
        } else if (kb == full && tail) {
          uint32_t b[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) b[j] = *reinterpret_cast<const uint32_t*>(us + 8 * j * a.u_row + 32 * kb + 4 * t);
#pragma unroll
          for (int m = 0; m < kM; ++m) {
            const uint8_t* t0 = ts + (rows_at + 16 * m + gid) * a.t_row + 32 * kb + 4 * t;
            const uint8_t* t1 = t0 + 8 * a.t_row;
            const uint32_t h0 = *reinterpret_cast<const uint32_t*>(t0), h1 = *reinterpret_cast<const uint32_t*>(t1);
            const uint32_t l0 = *reinterpret_cast<const uint32_t*>(t0 + width_t * 2), l1 = *reinterpret_cast<const uint32_t*>(t1 + width_t * 2);
#pragma unroll
            for (int j = 0; j < 4; ++j) ad_mma(d[m][j], h0, h1, l0, l1, b[j], b[j]);
          }
        }
      }
      const int col = now.col + 8 * t, left = now.end - col;  // this lane's columns
#pragma unroll
      for (int i = 0; i < 2 * kM; ++i) {
        if (rows[i] < 0) continue;
        const int m = i >> 1, h = 2 * (i & 1);
        const float f[8] = {d[m][0][h], d[m][0][h + 1], d[m][1][h], d[m][1][h + 1], d[m][2][h], d[m][2][h + 1], d[m][3][h], d[m][3][h + 1]};
        uint16_t* to = out + (long long)rows[i] * a.out_stride + col;
        if (a.vec && left >= 8) {
          float w[8];
          unpack8(v[i], w);
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] += f[e];
          st_vec(to, w);
        } else {
          const uint16_t* from = y + (long long)rows[i] * a.y_stride + col;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e < left) st_elem(to + e, ld_elem(from + e) + f[e]);
        }
      }
    }
    pair_sync();
    fetch_up(ring[kStages - 1], stage);
  }
  if constexpr (kRows == 16) ad_cluster_wait();
}

// ---------------------------------------------------------------------------------------------------------------- CUDA cores
// 32-bit models, and bf16 rows that cannot be read in 16 bytes: sixteen rows a cluster, 32-bit products.
constexpr int kAdSimtCluster = 8;

template <typename T>
__global__ void __launch_bounds__(kAdThreads) adapter_simt_kernel(const __grid_constant__ AdArgs a) {
  extern __shared__ __align__(16) uint8_t ad_smem[];
  constexpr int kC = kAdSimtCluster;
  const uint32_t smem = (uint32_t)__cvta_generic_to_shared(ad_smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = (int)ad_cluster_rank(), cl = blockIdx.x / kC;
  pdl_enter();
  pdl_wait();
  const int subs = a.tile_rows / 16;
  const int4 tile = a.tiles[cl / subs];
  const int32_t* order = a.order + (long long)cl * 16;
  const int slot = tile.x, count = min(tile.y - (cl % subs) * 16, 16);
  if (count <= 0) return;
  if (slot < 0) return ad_copy_rows<T, kC>(a, order, count, rank);
  const T* down = (const T*)a.down + (long long)slot * a.inner * a.width;
  const T* up = (const T*)a.up + (long long)slot * a.ends[a.parts - 1] * a.rank;
  float* part = reinterpret_cast<float*>(ad_smem);
  float* xs = part + 16 * a.inner_row;
  const int k0 = (int)((long long)a.width * rank / kC), k1 = (int)((long long)a.width * (rank + 1) / kC);
  for (int i = tid; i < 16 * a.inner_row; i += kAdThreads) part[i] = 0.f;
  for (int s0 = k0; s0 < k1; s0 += kAdSimtChannels) {
    const int n = min(k1 - s0, kAdSimtChannels);
    __syncthreads();
    for (int i = tid; i < 16 * kAdSimtChannels; i += kAdThreads) {
      const int row = i / kAdSimtChannels, k = i % kAdSimtChannels;
      xs[i] = row < count && k < n ? ld_elem((const T*)a.x + (long long)order[row] * a.x_stride + s0 + k) : 0.f;
    }
    __syncthreads();
    for (int j = warp; j < a.inner; j += kAdWarps) {
      float s[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = 0.f;
      for (int k = lane; k < n; k += 32) {
        const float w = ld_elem(down + (long long)j * a.width + s0 + k);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] += w * xs[r * kAdSimtChannels + k];
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float v = warp_sum(s[r]);
        if (lane == r) part[r * a.inner_row + j] += v;
      }
    }
  }
  ad_cluster_arrive();
  ad_cluster_wait();
  const int g0 = ad_first_group<kC>(a, rank), g1 = ad_first_group<kC>(a, rank + 1);
  const int p0 = g0 < g1 ? ad_group(a, g0).part : 0, quads = g0 < g1 ? ((ad_group(a, g1 - 1).part - p0 + 1) * a.rank) >> 2 : 0;
  const float scale = a.scale[slot];
  for (int i = tid; i < 16 * quads; i += kAdThreads) {
    const int row = i / quads, col = (i - row * quads) * 4;
    *reinterpret_cast<float4*>(ad_smem + a.off_t + row * a.t_row + col * 4) = ad_total<kC>(smem + (row * a.inner_row + p0 * a.rank + col) * 4, scale);
  }
  ad_cluster_arrive();
  __syncthreads();
  for (int g = g0 + warp; g < g1; g += kAdWarps) {
    const AdGroup gr = ad_group(a, g);
    const int col = gr.col + lane;
    if (col >= gr.end) continue;
    float d[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) d[r] = 0.f;
    const uint8_t* ts = ad_smem + a.off_t + (gr.part - p0) * a.rank * 4;
    for (int j = 0; j < a.rank; j += 4) {
      float u[4];
      ld_elem4(up + (long long)col * a.rank + j, u);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float4 v = *reinterpret_cast<const float4*>(ts + r * a.t_row + j * 4);
        d[r] += u[0] * v.x + u[1] * v.y + u[2] * v.z + u[3] * v.w;
      }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      if (r < count) {
        const long long row = order[r];
        st_elem((T*)a.out + row * a.out_stride + col, ld_elem((const T*)a.y + row * a.y_stride + col) + d[r]);
      }
    }
  }
  ad_cluster_wait();
}

// ---------------------------------------------------------------------------------------------------------------- launches
constexpr size_t kAdMostSmem = 220 * 1024;

template <typename... KArgs>
static int ad_launch(void (*kernel)(KArgs...), const AdArgs& a, int clusters, int cluster, size_t smem, cudaStream_t stream) {
  if (smem > kAdMostSmem) return B200KV_E_SHAPE;
  if (!allow_smem(kernel, kAdMostSmem)) return launch_result(cudaErrorInvalidValue);
  if (cluster > 8 && cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return launch_result(cudaErrorInvalidValue);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(clusters * cluster));
  cfg.blockDim = dim3(kAdThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = take_chained_launch(stream) ? 2 : 1;
  return launch_result(cudaLaunchKernelEx(&cfg, kernel, a));
}

// Most parts that the columns of one block touch.
static int ad_parts_spanned(const AdArgs& a, int cluster) {
  int most = 1;
  for (int q = 0; q < cluster; ++q) {
    const int g0 = (int)((unsigned)a.groups * (unsigned)q / cluster), g1 = (int)((unsigned)a.groups * (unsigned)(q + 1) / cluster);
    if (g0 >= g1) continue;
    int begin = 0, at = 0, lo = 0, hi = 0;
    for (int p = 0; p < a.parts; ++p) {
      const int n = (a.ends[p] - begin + 31) / 32;
      if (g0 >= at && g0 < at + n) lo = p;
      if (g1 - 1 >= at && g1 - 1 < at + n) hi = p;
      at += n;
      begin = a.ends[p];
    }
    if (hi - lo + 1 > most) most = hi - lo + 1;
  }
  return most;
}

template <int kRows, int kNT, int kKB, int kC, int kStages>
static int ad_run(AdArgs a, int clusters, cudaStream_t stream) {
  constexpr int kGroups = kRows == 16 ? 8 : 4;
  const int spanned = ad_parts_spanned(a, kC) * a.rank;
  a.inner_row = a.inner + 4;                    // (rows apart by other banks)
  a.t_row = (spanned * 4 + 63) / 64 * 64 + 32;  // both terms; four rows at different banks
  a.u_row = a.rank * 2;
  while (a.u_row % 64 != 32) a.u_row += 16;     // four columns at different banks
  size_t first;
  if (kRows == 16) {
    const int wn = (a.inner + 8 * kNT - 1) / (8 * kNT), deep = kAdWarps / (wn <= 1 ? 1 : (wn <= 2 ? 2 : (wn <= 4 ? 4 : 8)));
    first = (size_t)deep * 16 * a.inner_row * 4;
  } else {
    const size_t staged = (size_t)2 * a.inner * 128, partial = (size_t)kRows * a.inner_row * 4;
    first = staged > partial ? staged : partial;
  }
  a.off_t = (uint32_t)((first + 15) / 16 * 16);
  a.off_u = a.off_t + kRows * a.t_row;
  int stages = kStages;
  const int chunks = ((a.groups + kC - 1) / kC + kGroups - 1) / kGroups;  // of a block, at most
  if (stages > chunks) stages = chunks;
  return ad_launch(adapter_kernel<kRows, kNT, kKB, kC, kStages>, a, clusters, kC, a.off_u + (size_t)stages * kGroups * 32 * a.u_row, stream);
}

}  // namespace b200kv

using namespace b200kv;

extern "C" int b200dec_adapter_plan(const int32_t* ids, int32_t num_rows, int32_t slots, int32_t tile_rows, int32_t* order, int32_t* tiles,
                                    int32_t max_tiles, int32_t* status, void* stream) {
  if (num_rows == 0) return B200KV_OK;
  if (!ids || !order || !tiles) return B200KV_E_NULL;
  if (num_rows < 0 || num_rows > (1 << 26) || slots < 1 || slots > kAdMaxSlots) return B200KV_E_RANGE;
  if (tile_rows != 16 && tile_rows != 64) return B200KV_E_SHAPE;
  if (max_tiles < num_rows / tile_rows + (num_rows < slots + 1 ? num_rows : slots + 1)) return B200KV_E_WORKSPACE;
  if ((long long)max_tiles * tile_rows > 0x7fffffffLL) return B200KV_E_RANGE;
  if (!aligned(tiles, 16) || !aligned(ids, 4) || !aligned(order, 4)) return B200KV_E_ALIGN;
  const int threads = num_rows <= 256 && slots < 256 ? 256 : kAdPlanThreads;
  return launch_result(launch_chained(adapter_plan_kernel, dim3(1), dim3(threads), (size_t)(slots + 1) * 4, (cudaStream_t)stream, ids,
                                      (int)num_rows, (int)slots, (int)tile_rows, order, (int4*)tiles, (int)max_tiles, status));
}

extern "C" int b200dec_add_adapters(const b200dec_adapters* ad, const void* x, int64_t x_stride, const void* y, int64_t y_stride, void* out,
                                    int64_t out_stride, const int32_t* order, const int32_t* tiles, int32_t max_tiles, int32_t tile_rows,
                                    int32_t num_rows, void* stream) {
  if (num_rows == 0) return B200KV_OK;
  if (!ad || !ad->down || !ad->up || !ad->scale || !x || !y || !out || !order || !tiles) return B200KV_E_NULL;
  if (num_rows < 0 || max_tiles < 1 || ad->slots < 1 || ad->slots > kAdMaxSlots) return B200KV_E_RANGE;
  if (ad->elem != 2 && ad->elem != 4) return B200KV_E_SHAPE;
  if (ad->parts < 1 || ad->parts > kAdMaxParts || ad->rank < 8 || ad->rank > 128 || ad->rank % 8 || ad->width < 1) return B200KV_E_SHAPE;
  if (tile_rows != 16 && tile_rows != 64) return B200KV_E_SHAPE;
  AdArgs a = {};
  a.down = ad->down; a.up = ad->up; a.scale = ad->scale; a.x = x; a.y = y; a.out = out;
  a.x_stride = x_stride; a.y_stride = y_stride; a.out_stride = out_stride;
  a.order = order; a.tiles = (const int4*)tiles; a.tile_rows = tile_rows;
  a.rank = ad->rank; a.width = ad->width; a.parts = ad->parts;
  bool even = true;
  for (int p = 0, begin = 0; p < ad->parts; ++p) {
    if (ad->ends[p] <= begin || ad->ends[p] > (1 << 28)) return B200KV_E_SHAPE;
    even = even && begin % 8 == 0;
    a.ends[p] = ad->ends[p];
    a.groups += (ad->ends[p] - begin + 31) / 32;
    begin = ad->ends[p];
  }
  const int cols = a.ends[a.parts - 1];
  if (x_stride < a.width || y_stride < cols || out_stride < cols || out == x) return B200KV_E_SHAPE;
  if ((out == y && out_stride != y_stride) || (long long)max_tiles * tile_rows > 0x7fffffffLL) return B200KV_E_RANGE;
  if (!aligned(ad->down, 16) || !aligned(ad->up, 16) || !aligned(ad->scale, 4) || !aligned(tiles, 16) || !aligned(order, 4) || !aligned(x, ad->elem) ||
      !aligned(y, ad->elem) || !aligned(out, ad->elem))
    return B200KV_E_ALIGN;
  a.inner = a.parts * a.rank;
  a.vec = even && aligned(y, 16) && aligned(out, 16) && y_stride % 8 == 0 && out_stride % 8 == 0;
  cudaStream_t s = (cudaStream_t)stream;
  const int fine = max_tiles * (tile_rows / 16);  // clusters with sixteen rows each
  if (ad->elem == 4 || a.width % 8 || x_stride % 8 || !aligned(x, 16)) {
    a.inner_row = a.inner;
    a.t_row = ad_parts_spanned(a, kAdSimtCluster) * a.rank * 4;
    a.off_t = 16u * a.inner_row * 4 + 16u * kAdSimtChannels * 4;
    const size_t smem = a.off_t + (size_t)16 * a.t_row;
    return ad->elem == 4 ? ad_launch(adapter_simt_kernel<float>, a, fine, kAdSimtCluster, smem, s)
                         : ad_launch(adapter_simt_kernel<uint16_t>, a, fine, kAdSimtCluster, smem, s);
  }
  const int kb = (a.rank + 15) / 16;
  if (tile_rows == 16 || a.inner > kAdMaxInner) {
    if (kb <= 1) return ad_run<16, 4, 1, 8, 4>(a, fine, s);
    if (kb <= 2) return ad_run<16, 4, 2, 8, 4>(a, fine, s);
    if (kb <= 4) return ad_run<16, 4, 4, 8, 2>(a, fine, s);
    return ad_run<16, 8, 8, 8, 2>(a, fine, s);
  }
  if (kb <= 1) return ad_run<64, 8, 1, 8, 4>(a, max_tiles, s);
  if (kb <= 2) return ad_run<64, 16, 2, 8, 2>(a, max_tiles, s);
  if (kb <= 4) return ad_run<64, 24, 4, 8, 2>(a, max_tiles, s);
  return ad_run<64, 24, 8, 8, 2>(a, max_tiles, s);
}
