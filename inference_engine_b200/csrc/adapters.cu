// Low-rank adapters of many requests beside a shared projection:
//     out[r] = y[r] + scale[a] * (x[r] . down[a]^T) . up[a]^T,   a = the adapter of row r
// A packed projection has a `down` of its own for each part; a column of `up` meets the inner values of its part.
//
// The plan (one block, once per step) sorts the rows by adapter into tiles of at most `tile_rows` rows of one adapter.  A product is then
// one launch: a cluster of blocks takes a tile.  Its blocks share the input channels, so that a tile's `down` is fetched by many
// multiprocessors at once; their partial inner values are summed through distributed shared memory (every block sums some rows over all
// blocks, in a fixed order, and hands them to the blocks whose columns need them); then the blocks share the output columns.
//
// Precision: bf16 operands, 32-bit sums.  The inner values are scaled in 32 bits and enter the second product as two bf16 terms (16 bits of
// mantissa): rounded to one they would cost the sum as much as its own rounding does.
#include "dec_common.cuh"

namespace b200kv {

constexpr int kAdThreads = 256;
constexpr int kAdWarps = kAdThreads / 32;
constexpr int kAdCluster = 8;
constexpr int kAdMaxParts = 4;
constexpr int kAdMaxSlots = 4096;
constexpr int kAdPlanThreads = 1024;
constexpr int kAdSimtChannels = 512;  // input channels that the CUDA cores' form stages at a time

struct AdTile { int slot, first, count, unused; };

struct AdArgs {
  const void *down, *up;
  const float* scale;
  const void *x, *y;
  void* out;
  long long x_stride, y_stride, out_stride;
  const int32_t* order;
  const int4* tiles;
  int tile_rows;  // of the plan
  int slots, rank, width, parts, num_rows;
  int ends[kAdMaxParts];
  int groups;                   // of 32 output columns, none across parts
  int inner;                    // parts * rank
  int inner_row;                // floats between rows of partial inner values
  int t_row;                    // bytes between rows of finished ones
  int stage;                    // input channels staged at a time (tiles of 128 rows)
  int vec;                      // y and out rows can be read and written in 16 bytes
  uint32_t off_t;               // shared memory: the finished inner values
};

// ---------------------------------------------------------------------------------------------------------------- the plan
// Which rows of one adapter are where in `order` is left to atomics: a row's result does not depend on its place in a tile.
__global__ void __launch_bounds__(kAdPlanThreads)
adapter_plan_kernel(const int32_t* ids, int N, int slots, int tile_rows, int32_t* order, int4* tiles, int max_tiles, int32_t* status) {
  extern __shared__ int ad_plan_smem[];  // rows of each group, then where its next row goes; group `slots`: no adapter
  __shared__ int warp_rows[32], warp_tiles[32];
  pdl_enter();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int g = tid; g <= slots; g += kAdPlanThreads) ad_plan_smem[g] = 0;
  __syncthreads();
  auto group = [&](int r) {
    const int id = ids[r];
    if (id >= 0 && id < slots) return id;
    if (id != -1 && status) atomicOr(status, B200KV_S_BAD_POSITION);
    return slots;
  };
  for (int base = warp * 32; base < N; base += kAdPlanThreads) {
    const int r = base + lane;
    const unsigned on = __ballot_sync(0xffffffffu, r < N);
    if (r < N) {
      const int g = group(r);
      const unsigned same = __match_any_sync(on, g);
      if (lane == __ffs(same) - 1) atomicAdd(&ad_plan_smem[g], __popc(same));
    }
  }
  __syncthreads();
  int rows_before = 0, tiles_before = 0;
  for (int base = 0; base <= slots; base += kAdPlanThreads) {
    const int g = base + tid, n = g <= slots ? ad_plan_smem[g] : 0, t = (n + tile_rows - 1) / tile_rows;
    int rs = n, ts = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, rs, o), b = __shfl_up_sync(0xffffffffu, ts, o);
      if (lane >= o) { rs += a; ts += b; }
    }
    if (lane == 31) { warp_rows[warp] = rs; warp_tiles[warp] = ts; }
    __syncthreads();
    int rw = rows_before, tw = tiles_before, ra = 0, ta = 0;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) { rw += warp_rows[w]; tw += warp_tiles[w]; }
      ra += warp_rows[w];
      ta += warp_tiles[w];
    }
    const int first = rw + rs - n, tile = tw + ts - t;
    if (g <= slots) {
      ad_plan_smem[g] = first;
      for (int i = 0; i < t; ++i)
        if (tile + i < max_tiles) tiles[tile + i] = make_int4(g < slots ? g : -1, first + i * tile_rows, min(tile_rows, n - i * tile_rows), 0);
    }
    rows_before += ra;
    tiles_before += ta;
    __syncthreads();
  }
  for (int i = tiles_before + tid; i < max_tiles; i += kAdPlanThreads) tiles[i] = make_int4(-1, 0, 0, 0);
  for (int base = warp * 32; base < N; base += kAdPlanThreads) {
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
__device__ __forceinline__ void ad_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
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
__device__ __forceinline__ void ad_st_remote4(uint32_t addr, const float4& v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}

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
__device__ __forceinline__ int ad_first_group(const AdArgs& a, int rank) { return (int)((long long)a.groups * rank / kAdCluster); }

// Rows of the tile without an adapter: copied where the result has a place of its own.
template <typename T>
__device__ __forceinline__ void ad_copy_rows(const AdArgs& a, int first, int count, int rank) {
  if (a.out == a.y) return;
  const int lo = ad_first_group(a, rank), hi = ad_first_group(a, rank + 1);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int g = lo + warp; g < hi; g += kAdWarps) {
    const AdGroup gr = ad_group(a, g);
    if (gr.col + lane >= gr.end) continue;
    for (int i = 0; i < count; ++i) {
      const long long r = a.order[first + i];
      ((T*)a.out)[r * a.out_stride + gr.col + lane] = ((const T*)a.y)[r * a.y_stride + gr.col + lane];
    }
  }
}

// The finished inner values of this block's share of the tile's rows, over all blocks' partial ones (fp32 at offset 0, rows of a.inner_row
// floats), to every block whose columns need them (at a.off_t, rows of a.t_row bytes; columns from its first part on).
// kSplit: as two bf16 terms, the first ones of a row's columns before the second ones.
template <bool kSplit>
__device__ __forceinline__ void ad_exchange(const AdArgs& a, uint32_t smem, int rank, int rows, float scale) {
  const int quads = a.inner >> 2, n = rows * quads;
  for (int i = rank * kAdThreads + threadIdx.x; i < n; i += kAdCluster * kAdThreads) {
    const int row = i / quads, col = (i - row * quads) * 4;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    float4 v[kAdCluster];
#pragma unroll
    for (int q = 0; q < kAdCluster; ++q) v[q] = ad_ld_remote4(ad_at_rank(smem + (row * a.inner_row + col) * 4, q));
#pragma unroll
    for (int q = 0; q < kAdCluster; ++q) { s.x += v[q].x; s.y += v[q].y; s.z += v[q].z; s.w += v[q].w; }
    s.x *= scale; s.y *= scale; s.z *= scale; s.w *= scale;
    const int part = col / a.rank;
    uint32_t hi0 = 0, hi1 = 0, lo0 = 0, lo1 = 0;
    if constexpr (kSplit) {
      const uint32_t h[4] = {float_to_bf16_bits(s.x), float_to_bf16_bits(s.y), float_to_bf16_bits(s.z), float_to_bf16_bits(s.w)};
      hi0 = h[0] | (h[1] << 16);
      hi1 = h[2] | (h[3] << 16);
      // (an infinite or NaN value has no second term)
      const float f[4] = {s.x, s.y, s.z, s.w};
      uint32_t l[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float rest = f[j] - bf16_bits_to_float(h[j]);
        l[j] = fabsf(rest) < INFINITY ? float_to_bf16_bits(rest) : 0u;
      }
      lo0 = l[0] | (l[1] << 16);
      lo1 = l[2] | (l[3] << 16);
    }
#pragma unroll
    for (int q = 0; q < kAdCluster; ++q) {
      const int g0 = ad_first_group(a, q), g1 = ad_first_group(a, q + 1);
      if (g0 >= g1) continue;
      const int p0 = ad_group(a, g0).part, p1 = ad_group(a, g1 - 1).part;
      if (part < p0 || part > p1) continue;
      const int at = col - p0 * a.rank;
      if constexpr (kSplit) {
        const uint32_t dst = ad_at_rank(smem + a.off_t + row * a.t_row + at * 2, q);
        ad_st_remote2(dst, hi0, hi1);
        ad_st_remote2(dst + (p1 - p0 + 1) * a.rank * 2, lo0, lo1);
      } else {
        ad_st_remote4(ad_at_rank(smem + a.off_t + row * a.t_row + at * 4, q), s);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------- tensor cores
// kRows 16: the warps share the block's channels and, where there are more than 64 inner values, those too; both operands go straight
// from memory to registers.  kRows 128: a warp takes sixteen rows, `down` is staged in shared memory for all of them.
// kNT: blocks of eight inner values of a warp.  kKB: blocks of sixteen inner values of a part.
// The order of a product's channels is free, so that a lane loads whole 16 bytes: lane t of a row's four has channels 8t .. 8t + 7 of 32.
template <int kRows, int kNT, int kKB>
__global__ void __launch_bounds__(kAdThreads) adapter_kernel(const __grid_constant__ AdArgs a) {
  extern __shared__ __align__(16) uint8_t ad_smem[];
  const uint32_t smem = (uint32_t)__cvta_generic_to_shared(ad_smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, t = lane & 3;
  const int rank = (int)ad_cluster_rank(), cl = blockIdx.x / kAdCluster;
  pdl_enter();
  pdl_wait();
  const int subs = a.tile_rows / kRows, sub = subs > 1 ? cl % subs : 0;
  const int4 tile = a.tiles[subs > 1 ? cl / subs : cl];
  const int slot = tile.x, first = tile.y + sub * kRows, count = min(tile.z - sub * kRows, kRows);
  if (count <= 0) return;  // (with the whole cluster)
  if (slot < 0) return ad_copy_rows<uint16_t>(a, first, count, rank);
  const uint16_t* down = (const uint16_t*)a.down + (long long)slot * a.inner * a.width;
  const uint16_t* up = (const uint16_t*)a.up + (long long)slot * a.ends[a.parts - 1] * a.rank;
  const uint4 zero4 = make_uint4(0, 0, 0, 0);
  const int chunks = (a.width + 31) >> 5;
  float* part = reinterpret_cast<float*>(ad_smem);

  float acc[kNT][4];
#pragma unroll
  for (int n = 0; n < kNT; ++n)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[n][j] = 0.f;
  const int m0 = kRows == 16 ? 0 : 16 * warp;
  const int r0 = m0 + gid, r1 = r0 + 8;
  const uint16_t* x0 = (const uint16_t*)a.x + (r0 < count ? (long long)a.order[first + r0] * a.x_stride : 0);
  const uint16_t* x1 = (const uint16_t*)a.x + (r1 < count ? (long long)a.order[first + r1] * a.x_stride : 0);

  if constexpr (kRows == 16) {
    const int wn = (a.inner + 8 * kNT - 1) / (8 * kNT);                // warps side by side over the inner values
    const int across = wn <= 1 ? 1 : (wn <= 2 ? 2 : (wn <= 4 ? 4 : 8)), deep = kAdWarps / across;
    const int n0 = (warp % across) * kNT * 8, d = warp / across;
    for (int c = rank * deep + d; c < chunks; c += kAdCluster * deep) {
      const int k = 32 * c + 8 * t;
      const bool in = k < a.width;  // (a multiple of 8)
      const uint4 u0 = in && r0 < count ? *reinterpret_cast<const uint4*>(x0 + k) : zero4;
      const uint4 u1 = in && r1 < count ? *reinterpret_cast<const uint4*>(x1 + k) : zero4;
      uint4 w[kNT];
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        const int j = n0 + 8 * n + gid;
        w[n] = in && j < a.inner ? __ldg(reinterpret_cast<const uint4*>(down + (long long)j * a.width + k)) : zero4;
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
    const int c0 = chunks * rank / kAdCluster, c1 = chunks * (rank + 1) / kAdCluster;
    const int row_bytes = a.stage * 2 + (a.stage % 64 == 0 ? 64 : 0);  // two rows apart by half a line of banks
    for (int s0 = c0; s0 < c1; s0 += a.stage / 32) {
      const int s1 = min(c1, s0 + a.stage / 32), vecs = (s1 - s0) * 4;
      if (s0 > c0) __syncthreads();
      for (int i = tid; i < a.inner * vecs; i += kAdThreads) {
        const int j = i / vecs, v = i - j * vecs, k = 32 * s0 + 8 * v;
        const uint32_t dst = smem + j * row_bytes + v * 16;
        const int bytes = k < a.width ? 16 : 0;  // what lies behind the width is zero
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(down + (bytes ? (long long)j * a.width + k : 0)), "r"(bytes) : "memory");
      }
      asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;\n" ::: "memory");
      __syncthreads();
      if (m0 < count) {
#pragma unroll 2
        for (int c = s0; c < s1; ++c) {
          const int k = 32 * c + 8 * t;
          const bool in = k < a.width;
          const uint4 u0 = in && r0 < count ? *reinterpret_cast<const uint4*>(x0 + k) : zero4;
          const uint4 u1 = in && r1 < count ? *reinterpret_cast<const uint4*>(x1 + k) : zero4;
#pragma unroll
          for (int n = 0; n < kNT; ++n) {
            if (8 * n < a.inner) {
              const uint4 w = *reinterpret_cast<const uint4*>(ad_smem + (8 * n + gid) * row_bytes + (c - s0) * 64 + t * 16);
              ad_mma(acc[n], u0.x, u1.x, u0.y, u1.y, w.x, w.y);
              ad_mma(acc[n], u0.z, u1.z, u0.w, u1.w, w.z, w.w);
            }
          }
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
      const int j = 8 * n + 2 * t;
      if (8 * n < a.inner && m0 < count) {
        *reinterpret_cast<float2*>(part + r0 * a.inner_row + j) = make_float2(acc[n][0], acc[n][1]);
        *reinterpret_cast<float2*>(part + r1 * a.inner_row + j) = make_float2(acc[n][2], acc[n][3]);
      }
    }
  }
  ad_cluster_sync();
  ad_exchange<true>(a, smem, rank, count, a.scale[slot]);
  ad_cluster_sync();  // nobody reads another block's memory behind this

  // ---- the second product: 32 columns of a warp at a time, as four tiles of eight.  Tile j's column n is column 8 (n / 2) + 2 j + n % 2 of the 32, so that a
  // lane has eight columns side by side.  Lane t of a row's four has inner values 4t .. 4t + 3 of sixteen; where eight are left over, the two
  // terms of 2t and 2t + 1 share one step.
  const int g0 = ad_first_group(a, rank), g1 = ad_first_group(a, rank + 1);
  if (g0 >= g1) return;
  const int p0 = ad_group(a, g0).part, width_t = (ad_group(a, g1 - 1).part - p0 + 1) * a.rank;
  const int full = a.rank >> 4;
  const bool tail = a.rank & 8;
  const uint8_t* ts = ad_smem + a.off_t;
  const uint16_t* y = (const uint16_t*)a.y;
  uint16_t* out = (uint16_t*)a.out;
  for (int g = g0 + warp; g < g1; g += kAdWarps) {
    const AdGroup gr = ad_group(a, g);
    uint2 b[kKB][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int col = min(gr.col + 8 * (gid >> 1) + 2 * j + (gid & 1), gr.end - 1);
      const uint16_t* u = up + (long long)col * a.rank;
#pragma unroll
      for (int kb = 0; kb < kKB; ++kb) {
        if (kb < full) {
          b[kb][j] = __ldg(reinterpret_cast<const uint2*>(u + 16 * kb + 4 * t));
        } else if (kb == full && tail) {
          const uint32_t v = __ldg(reinterpret_cast<const uint32_t*>(u + 16 * kb + 2 * t));
          b[kb][j] = make_uint2(v, v);
        }
      }
    }
    const int col = gr.col + 8 * t, left = gr.end - col;  // this lane's columns
    const bool whole = a.vec && left >= 8;
    for (int m = 0; m < count; m += 16) {
      const int ra = m + gid, rb = ra + 8;
      const long long ya = ra < count ? (long long)a.order[first + ra] : -1, yb = rb < count ? (long long)a.order[first + rb] : -1;
      uint4 va = zero4, vb = zero4;
      if (whole) {
        if (ya >= 0) va = *reinterpret_cast<const uint4*>(y + ya * a.y_stride + col);
        if (yb >= 0) vb = *reinterpret_cast<const uint4*>(y + yb * a.y_stride + col);
      }
      float d[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) d[j][i] = 0.f;
      const uint8_t* ta = ts + ra * a.t_row + (gr.part - p0) * a.rank * 2;
      const uint8_t* tb = ta + 8 * a.t_row;
#pragma unroll
      for (int kb = 0; kb < kKB; ++kb) {
        if (kb < full) {
          const uint2 h0 = *reinterpret_cast<const uint2*>(ta + 32 * kb + 8 * t), h1 = *reinterpret_cast<const uint2*>(tb + 32 * kb + 8 * t);
          const uint2 l0 = *reinterpret_cast<const uint2*>(ta + width_t * 2 + 32 * kb + 8 * t), l1 = *reinterpret_cast<const uint2*>(tb + width_t * 2 + 32 * kb + 8 * t);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            ad_mma(d[j], h0.x, h1.x, h0.y, h1.y, b[kb][j].x, b[kb][j].y);
            ad_mma(d[j], l0.x, l1.x, l0.y, l1.y, b[kb][j].x, b[kb][j].y);
          }
        } else if (kb == full && tail) {
          const uint32_t h0 = *reinterpret_cast<const uint32_t*>(ta + 32 * kb + 4 * t), h1 = *reinterpret_cast<const uint32_t*>(tb + 32 * kb + 4 * t);
          const uint32_t l0 = *reinterpret_cast<const uint32_t*>(ta + width_t * 2 + 32 * kb + 4 * t), l1 = *reinterpret_cast<const uint32_t*>(tb + width_t * 2 + 32 * kb + 4 * t);
#pragma unroll
          for (int j = 0; j < 4; ++j) ad_mma(d[j], h0, h1, l0, l1, b[kb][j].x, b[kb][j].y);
        }
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const long long row = half ? yb : ya;
        if (row < 0) continue;
        const float f[8] = {d[0][2 * half], d[0][2 * half + 1], d[1][2 * half], d[1][2 * half + 1], d[2][2 * half], d[2][2 * half + 1], d[3][2 * half], d[3][2 * half + 1]};
        if (whole) {
          float v[8];
          unpack8(half ? vb : va, v);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] += f[i];
          st_vec(out + row * a.out_stride + col, v);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (i < left) st_elem(out + row * a.out_stride + col + i, ld_elem(y + row * a.y_stride + col + i) + f[i]);
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------- CUDA cores
// 32-bit models, and bf16 rows that cannot be read in 16 bytes: sixteen rows a cluster, 32-bit products.
template <typename T>
__global__ void __launch_bounds__(kAdThreads) adapter_simt_kernel(const __grid_constant__ AdArgs a) {
  extern __shared__ __align__(16) uint8_t ad_smem[];
  const uint32_t smem = (uint32_t)__cvta_generic_to_shared(ad_smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = (int)ad_cluster_rank(), cl = blockIdx.x / kAdCluster;
  pdl_enter();
  pdl_wait();
  const int subs = a.tile_rows / 16, sub = cl % subs;
  const int4 tile = a.tiles[cl / subs];
  const int slot = tile.x, first = tile.y + sub * 16, count = min(tile.z - sub * 16, 16);
  if (count <= 0) return;
  if (slot < 0) return ad_copy_rows<T>(a, first, count, rank);
  const T* down = (const T*)a.down + (long long)slot * a.inner * a.width;
  const T* up = (const T*)a.up + (long long)slot * a.ends[a.parts - 1] * a.rank;
  float* part = reinterpret_cast<float*>(ad_smem);
  float* xs = part + 16 * a.inner_row;
  const int k0 = (int)((long long)a.width * rank / kAdCluster), k1 = (int)((long long)a.width * (rank + 1) / kAdCluster);
  for (int i = tid; i < 16 * a.inner_row; i += kAdThreads) part[i] = 0.f;
  for (int s0 = k0; s0 < k1; s0 += kAdSimtChannels) {
    const int n = min(k1 - s0, kAdSimtChannels);
    __syncthreads();
    for (int i = tid; i < 16 * kAdSimtChannels; i += kAdThreads) {
      const int row = i / kAdSimtChannels, k = i % kAdSimtChannels;
      xs[i] = row < count && k < n ? ld_elem((const T*)a.x + (long long)a.order[first + row] * a.x_stride + s0 + k) : 0.f;
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
  ad_cluster_sync();
  ad_exchange<false>(a, smem, rank, count, a.scale[slot]);
  ad_cluster_sync();
  const int g0 = ad_first_group(a, rank), g1 = ad_first_group(a, rank + 1);
  if (g0 >= g1) return;
  const int p0 = ad_group(a, g0).part;
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
        const long long row = a.order[first + r];
        st_elem((T*)a.out + row * a.out_stride + col, ld_elem((const T*)a.y + row * a.y_stride + col) + d[r]);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------- launches
constexpr size_t kAdMostSmem = 220 * 1024;

template <typename... KArgs>
static int ad_launch(void (*kernel)(KArgs...), const AdArgs& a, int clusters, size_t smem, cudaStream_t stream) {
  if (!allow_smem(kernel, kAdMostSmem)) return launch_result(cudaErrorInvalidValue);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)clusters * kAdCluster);
  cfg.blockDim = dim3(kAdThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kAdCluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = take_chained_launch(stream) ? 2 : 1;
  return launch_result(cudaLaunchKernelEx(&cfg, kernel, a));
}

// Most parts that the columns of one block touch.
static int ad_parts_spanned(const AdArgs& a) {
  int most = 1;
  for (int q = 0; q < kAdCluster; ++q) {
    const int g0 = (int)((long long)a.groups * q / kAdCluster), g1 = (int)((long long)a.groups * (q + 1) / kAdCluster);
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

}  // namespace b200kv

using namespace b200kv;

extern "C" int b200dec_adapter_plan(const int32_t* ids, int32_t num_rows, int32_t slots, int32_t tile_rows, int32_t* order, int32_t* tiles,
                                    int32_t max_tiles, int32_t* status, void* stream) {
  if (num_rows == 0) return B200KV_OK;
  if (!ids || !order || !tiles) return B200KV_E_NULL;
  if (num_rows < 0 || slots < 1 || slots > kAdMaxSlots) return B200KV_E_RANGE;
  if (tile_rows != 16 && tile_rows != 128) return B200KV_E_SHAPE;
  if (max_tiles < num_rows / tile_rows + (num_rows < slots + 1 ? num_rows : slots + 1)) return B200KV_E_WORKSPACE;
  if (!aligned(tiles, 16) || !aligned(ids, 4) || !aligned(order, 4)) return B200KV_E_ALIGN;
  return launch_result(launch_chained(adapter_plan_kernel, dim3(1), dim3(kAdPlanThreads), (size_t)(slots + 1) * 4, (cudaStream_t)stream, ids,
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
  if (tile_rows != 16 && tile_rows != 128) return B200KV_E_SHAPE;
  AdArgs a = {};
  a.down = ad->down; a.up = ad->up; a.scale = ad->scale; a.x = x; a.y = y; a.out = out;
  a.x_stride = x_stride; a.y_stride = y_stride; a.out_stride = out_stride;
  a.order = order; a.tiles = (const int4*)tiles; a.tile_rows = tile_rows;
  a.slots = ad->slots; a.rank = ad->rank; a.width = ad->width; a.parts = ad->parts; a.num_rows = num_rows;
  bool even = true;
  for (int p = 0, begin = 0; p < ad->parts; ++p) {
    if (ad->ends[p] <= begin) return B200KV_E_SHAPE;
    even = even && begin % 8 == 0;
    a.ends[p] = ad->ends[p];
    a.groups += (ad->ends[p] - begin + 31) / 32;
    begin = ad->ends[p];
  }
  const int cols = a.ends[a.parts - 1];
  if (x_stride < a.width || y_stride < cols || out_stride < cols) return B200KV_E_SHAPE;
  if ((out == y && out_stride != y_stride) || (long long)max_tiles * kAdCluster * (tile_rows / 16) > 0x7fffffffLL) return B200KV_E_RANGE;
  if (!aligned(ad->down, 16) || !aligned(ad->up, 16) || !aligned(ad->scale, 4) || !aligned(tiles, 16) || !aligned(order, 4) || !aligned(x, ad->elem) ||
      !aligned(y, ad->elem) || !aligned(out, ad->elem))
    return B200KV_E_ALIGN;
  a.inner = a.parts * a.rank;
  a.vec = even && aligned(y, 16) && aligned(out, 16) && y_stride % 8 == 0 && out_stride % 8 == 0;
  const int spanned = ad_parts_spanned(a) * a.rank;
  cudaStream_t s = (cudaStream_t)stream;
  const int fine = max_tiles * (tile_rows / 16);  // clusters with sixteen rows each
  if (ad->elem == 4 || a.width % 8 || x_stride % 8 || !aligned(x, 16)) {
    a.inner_row = a.inner;
    a.t_row = spanned * 4;
    a.off_t = 16u * a.inner_row * 4 + 16u * kAdSimtChannels * 4;
    const size_t smem = a.off_t + (size_t)16 * a.t_row;
    return ad->elem == 4 ? ad_launch(adapter_simt_kernel<float>, a, fine, smem, s) : ad_launch(adapter_simt_kernel<uint16_t>, a, fine, smem, s);
  }
  a.inner_row = a.inner + 4;               // (rows apart by other banks)
  a.t_row = (spanned * 4 + 63) / 64 * 64 + 32;  // both terms; four rows on different banks
  const int kb = (a.rank + 15) / 16;
  if (tile_rows == 16 || a.inner > 192) {
    const int wn = (a.inner + 63) / 64, deep = kAdWarps / (wn <= 1 ? 1 : (wn <= 2 ? 2 : (wn <= 4 ? 4 : 8)));
    a.off_t = ((uint32_t)deep * 16 * a.inner_row * 4 + 15) / 16 * 16;
    const size_t smem = a.off_t + (size_t)16 * a.t_row;
    if (kb <= 1) return ad_launch(adapter_kernel<16, 8, 1>, a, fine, smem, s);
    if (kb <= 2) return ad_launch(adapter_kernel<16, 8, 2>, a, fine, smem, s);
    if (kb <= 4) return ad_launch(adapter_kernel<16, 8, 4>, a, fine, smem, s);
    return ad_launch(adapter_kernel<16, 8, 8>, a, fine, smem, s);
  }
  // as many channels at a time as a block has, in 96 KB at most
  const int share = ((a.width + 31) / 32 + kAdCluster - 1) / kAdCluster * 32;
  int stage = 96 * 1024 / (a.inner * 2) / 32 * 32;
  a.stage = stage < share ? stage : share;
  const size_t staged = (size_t)a.inner * (a.stage * 2 + (a.stage % 64 == 0 ? 64 : 0)), partial = (size_t)128 * a.inner_row * 4;
  a.off_t = (uint32_t)(((staged > partial ? staged : partial) + 15) / 16 * 16);
  const size_t smem = a.off_t + (size_t)128 * a.t_row;
  if (smem > kAdMostSmem) return B200KV_E_SHAPE;
  if (kb <= 1) return ad_launch(adapter_kernel<128, 8, 1>, a, max_tiles, smem, s);
  if (kb <= 2) return ad_launch(adapter_kernel<128, 16, 2>, a, max_tiles, smem, s);
  if (kb <= 4) return ad_launch(adapter_kernel<128, 24, 4>, a, max_tiles, smem, s);
  return ad_launch(adapter_kernel<128, 24, 8>, a, max_tiles, smem, s);
}
