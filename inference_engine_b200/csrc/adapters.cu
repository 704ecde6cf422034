// Low-rank adapters of many requests beside a shared projection:
//     out[r] = y[r] + scale[a] * (x[r] . down[a]^T) . up[a]^T,   a = the adapter of row r
// A packed projection has a `down` of its own for each part; a column of `up` meets the inner values of its part.
//
// The plan (one block, once per step) sorts the rows by adapter into tiles of at most `tile_rows` rows of one adapter.  The products have a form for
// few rows of an adapter, where its weights are what is read (sixteen rows, mma.sync, one launch), one for portions, where x, y and the result
// are (128 rows, tcgen05, two launches), and one for rows on the CUDA cores.  In all, a cluster of blocks takes a tile and shares its input channels, so
// that a tile's `down` is fetched by many multiprocessors at once; the blocks' partial inner values are summed through distributed shared memory, in a fixed
// order.
//
// Precision: bf16 operands, 32-bit sums.  The inner values are scaled in 32 bits and enter the second product as two bf16 terms, which leave out 2^-16 of each
// at most: rounded to one they would cost the sum as much as its own rounding does, and with all of their bits a result comes out
// otherwise for one element in a thousand, by a last bit of its own (as near to the formula in 64 bits).  On the CUDA cores they keep their 32 bits.
//
// Measured, the plan and [2048 -> 4096] (three parts), [2048 -> 2048], [2048 -> 12288] (two parts) and [6144 -> 2048] in turn: one row, rank 16, 3.0 and 4.0,
// 4.0, 5.4 and 4.9 us; 64 rows of 48 adapters of rank 16 3.6 and 8.3, 6.6, 12.4 (28 MB, 2.3 TB/s) and 7.8; 992 rows of 3 adapters of rank 16 3.9 and 11, 7,
// 19 and 9; 2000 rows of 4 adapters of rank 64 4.7 and 26, 17, 38 (115 MB, 3 TB/s) and 25.  What bounds the small ones is a chain of latencies: tile, rows,
// first product, exchange, second product, result.
#include "dec_tma.cuh"

#include <algorithm>

namespace b200kv {

constexpr int kAdThreads = 256;
constexpr int kAdWarps = kAdThreads / 32;
constexpr int kAdMaxParts = 4;
constexpr int kAdMaxSlots = 4096;
constexpr int kAdPlanThreads = 512;
constexpr int kAdPlanAhead = 4;       // rows whose adapters a thread of the plan fetches together
constexpr int kAdSimtChannels = kAdThreads;  // input channels that the CUDA cores' form stages at a time
constexpr int kAdSimtCluster = 8;
constexpr int kAdTcCols = 128;        // output columns of a product of the tensor core
constexpr int kAdSecondThreads = 320;

struct AdArgs {
  const void *down, *up;
  const float* scale;
  const void *x, *y;
  void* out;
  long long x_stride, y_stride, out_stride;
  const int32_t* order;
  const int4* tiles;
  int tile_rows, max_tiles;  // of the plan
  int rank, width, parts;
  int ends[kAdMaxParts];
  int inner_row;          // floats between rows of partial inner values
  int t_row;              // bytes between rows of finished ones
  int u_row;              // bytes between columns of `up` in shared memory
  int ring;               // groups of columns on their way that a warp has room for
  int vec;                // y and out rows can be read and written in 16 bytes
  uint32_t off_t, off_u;  // shared memory: the finished inner values, `up`
  int32_t* status;
  // tiles of 128 rows
  void* terms;            // [tile][part][blocks of 64 inner values, both terms][128 rows of 128 bytes]: the second product's operand
  int blocks;
  int group_parts, part_groups;  // parts of a cluster of the first product
  uint32_t tmem_cols;
  int col_blocks, room;   // of the second product: all parts' blocks of columns, blocks that are resident at once
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
  // f(row, its adapter, the warp's lanes with a row) of all rows
  auto each = [&](auto f) {
    for (int base = tid; base - lane < N; base += kAdPlanAhead * threads) {
      int id[kAdPlanAhead];
#pragma unroll
      for (int j = 0; j < kAdPlanAhead; ++j) id[j] = base + j * threads < N ? ld_fresh(ids + base + j * threads) : -1;
#pragma unroll
      for (int j = 0; j < kAdPlanAhead; ++j) {
        const int r = base + j * threads;
        const unsigned on = __ballot_sync(0xffffffffu, r < N);
        if (r < N) f(r, id[j], on);
      }
    }
  };
  each([&](int, int id, unsigned on) {
    const bool known = id >= 0 && id < slots;
    if (!known && id != -1 && status) atomicOr(status, B200KV_S_BAD_POSITION);
    const int g = known ? id : slots;
    const unsigned same = __match_any_sync(on, g);
    if (lane == __ffs(same) - 1) atomicAdd(&ad_plan_smem[g], __popc(same));
  });
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
  if (tid == 0) tiles[0].z = tiles_before;  // (there is a row; its tile was written before the last barrier)
  each([&](int r, int id, unsigned on) {
    const int g = id >= 0 && id < slots ? id : slots;
    const unsigned same = __match_any_sync(on, g);
    int at = 0;
    if (lane == __ffs(same) - 1) at = atomicAdd(&ad_plan_smem[g], __popc(same));
    at = __shfl_sync(same, at, __ffs(same) - 1);
    order[at + __popc(same & ((1u << lane) - 1))] = r;
  });
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
__device__ __forceinline__ void ad_st_remote2(uint32_t addr, const uint2& v) {
  asm volatile("st.shared::cluster.v2.b32 [%0], {%1,%2};" ::"r"(addr), "r"(v.x), "r"(v.y) : "memory");
}
__device__ __forceinline__ void ad_copy16(uint32_t dst, const void* src, int bytes) {  // zeros behind the first `bytes`
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void ad_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void ad_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(kLeft) : "memory"); }

// Tiles, rows' places, x and y are read through L2.  A chained kernel is brought up beside the two or three in front of it: the multiprocessor's L1 may hold
// lines of theirs that were read before others wrote them (an older plan at the same address, say), and keeps none of what this one reads for the next.
// The rows [first, first + n) of a cluster's tile and the columns of its part.
struct AdJob {
  int slot, count, part, begin, end;
  const int32_t* order;
};
template <int kRows, int kC>
__device__ __forceinline__ AdJob ad_job(const AdArgs& a) {
  const int subs = a.tile_rows / kRows, cl = blockIdx.x / kC, at = cl / a.parts, part = cl - at * a.parts;
  const int4 tile = __ldcg(a.tiles + at / subs);
  return {tile.x, min(tile.y - (at % subs) * kRows, kRows), part, part ? a.ends[part - 1] : 0, a.ends[part], a.order + (long long)at * kRows};
}

// Rows without an adapter: copied where the result has a place of its own, sixteen at a time (lane i % 16 has row i) so that their loads are on their way together.
template <typename T>
__device__ __forceinline__ void ad_copy_rows(const AdArgs& a, int lane_row, int count, int col, int end, int step) {
  for (; __any_sync(0xffffffffu, col < end); col += step) {
    T v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = __shfl_sync(0xffffffffu, lane_row, i);
      if (i < count && col < end) v[i] = __ldcg((const T*)a.y + r * a.y_stride + col);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = __shfl_sync(0xffffffffu, lane_row, i);
      if (i < count && col < end) ((T*)a.out)[r * a.out_stride + col] = v[i];
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

__device__ __forceinline__ uint32_t ad_pack(float lo, float hi) {
  uint32_t v;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
  return v;
}
// What a lane adds to its eight columns of a row, f, which start `left` columns in front of the part's end; v: y's where `whole`.
__device__ __forceinline__ void ad_store(const uint16_t* from, uint16_t* to, int left, bool whole, const uint4& v, const float (&f)[8]) {
  if (whole) {
    float w[8];
    unpack8(v, w);
    uint4 o;
    o.x = ad_pack(w[0] + f[0], w[1] + f[1]);
    o.y = ad_pack(w[2] + f[2], w[3] + f[3]);
    o.z = ad_pack(w[4] + f[4], w[5] + f[5]);
    o.w = ad_pack(w[6] + f[6], w[7] + f[7]);
    *reinterpret_cast<uint4*>(to) = o;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < left) st_elem(to + e, ld_fresh(from + e) + f[e]);
  }
}

// ---------------------------------------------------------------------------------------------------------------- few rows: mma.sync
// The warps share the block's channels and, where there are more than 64 inner values, those too; both operands go straight from memory to
// registers.  The order of a product's channels is free, so that a lane loads whole 16 bytes: lane t of a row's four has channels 8t ..
// 8t + 7 of 32.  Second product: a warp takes groups of 32 columns, whose `up` and y come through a ring of its own.
// kNT: blocks of eight inner values of a warp.  kKB: blocks of sixteen inner values.  kC: blocks of a cluster.  kStages: groups on their way.
// Blocks that a multiprocessor's registers are shared among.  Three (80 registers) spilled above rank 32, where shared memory has room for one or two for the
// most part: one row of rank 64 beside [2048 -> 12288] 9.4 us, and 8.6 so.
constexpr int ad_rows_blocks(int inner_blocks) { return inner_blocks > 4 ? 1 : inner_blocks > 2 ? 2 : 3; }

template <int kNT, int kKB, int kC, int kStages>
__global__ void __launch_bounds__(kAdThreads, ad_rows_blocks(kKB)) adapter_rows_kernel(const __grid_constant__ AdArgs a) {
  extern __shared__ __align__(16) uint8_t ad_smem[];
  const uint32_t smem = (uint32_t)__cvta_generic_to_shared(ad_smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, t = lane & 3;
  const int rank = (int)ad_cluster_rank();
  pdl_enter();
  pdl_wait();
  const AdJob job = ad_job<16, kC>(a);
  const int lane_row = ld_fresh(job.order + (lane & 15));
  const int row0 = __shfl_sync(0xffffffffu, lane_row, gid), row1 = __shfl_sync(0xffffffffu, lane_row, gid + 8);
  if (job.count <= 0) return;  // (with the whole cluster)
  if (job.slot < 0) {
    if (a.out != a.y) ad_copy_rows<uint16_t>(a, lane_row, job.count, job.begin + rank * kAdThreads + tid, job.end, kC * kAdThreads);
    return;
  }
  const uint16_t* down = (const uint16_t*)a.down + ((long long)job.slot * a.parts + job.part) * a.rank * a.width;
  const uint16_t* up = (const uint16_t*)a.up + (long long)job.slot * a.ends[a.parts - 1] * a.rank;
  const uint16_t* y = (const uint16_t*)a.y;
  const uint4 zero4 = make_uint4(0, 0, 0, 0);
  const int chunks = (a.width + 31) >> 5;
  float* part = reinterpret_cast<float*>(ad_smem);
  const int groups = (job.end - job.begin + 31) >> 5, g0 = groups * rank / kC, g1 = groups * (rank + 1) / kC;

  // A stage: 32 columns of `up`, column 8 (n / 2) + 2 j + n % 2 at 8 j + n (see below), and what this lane needs of y.
  const int vecs = a.rank >> 3, stage_bytes = 32 * a.u_row + 1024;
  const uint32_t ring = a.off_u + warp * a.ring * stage_bytes;
  const unsigned by_vecs = (65536u + vecs - 1) / vecs;  // i / vecs of i < 512 by a product
  auto fetch = [&](int g, int stage) {
    if (g < g1) {
      const int col0 = job.begin + 32 * g, left = job.end - col0;
      const uint16_t* src = up + (long long)col0 * a.rank;
      const uint32_t dst = smem + ring + stage * stage_bytes;
      for (int i = lane; i < 32 * vecs; i += 32) {
        const int c = (int)((unsigned)i * by_vecs >> 16), v = i - c * vecs;
        const int place = 8 * ((c >> 1) & 3) + 2 * (c >> 3) + (c & 1);
        ad_copy16(dst + place * a.u_row + v * 16, c < left ? src + i * 8 : up, c < left ? 16 : 0);
      }
      const bool whole = a.vec && left - 8 * t >= 8;
      const uint32_t ydst = dst + 32 * a.u_row + lane * 16;
      if (whole && row0 >= 0) ad_copy16(ydst, y + (long long)row0 * a.y_stride + col0 + 8 * t, 16);
      if (whole && row1 >= 0) ad_copy16(ydst + 512, y + (long long)row1 * a.y_stride + col0 + 8 * t, 16);
    }
    ad_commit();
  };

  float acc[kNT][4];
#pragma unroll
  for (int n = 0; n < kNT; ++n)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[n][j] = 0.f;
  const uint16_t* x0 = (const uint16_t*)a.x + (long long)max(row0, 0) * a.x_stride;
  const uint16_t* x1 = (const uint16_t*)a.x + (long long)max(row1, 0) * a.x_stride;
  const int across = a.rank <= 8 * kNT ? 1 : 2, deep = kAdWarps / across;  // warps side by side over the inner values
  const int n0 = (warp % across) * kNT * 8, d = warp / across;
  bool first = true;
  for (int c = rank * deep + d; c < chunks || first; c += kC * deep) {
    const int k = 32 * c + 8 * t;  // (the width is a multiple of 8)
    const bool in = k < a.width;
    uint4 w[kNT];
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
      const int j = n0 + 8 * n + gid;
      w[n] = in && j < a.rank ? __ldg(reinterpret_cast<const uint4*>(down + (long long)j * a.width + k)) : zero4;
    }
    const uint4 u0 = in && row0 >= 0 ? __ldcg(reinterpret_cast<const uint4*>(x0 + k)) : zero4;
    const uint4 u1 = in && row1 >= 0 ? __ldcg(reinterpret_cast<const uint4*>(x1 + k)) : zero4;
    if (first) {
#pragma unroll
      for (int i = 0; i < kStages; ++i) fetch(g0 + warp + i * kAdWarps, i);
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
    if (j < a.rank) {
      *reinterpret_cast<float2*>(mine + gid * a.inner_row + j) = make_float2(acc[n][0], acc[n][1]);
      *reinterpret_cast<float2*>(mine + (gid + 8) * a.inner_row + j) = make_float2(acc[n][2], acc[n][3]);
    }
  }
  __syncthreads();
  const int quads = a.rank >> 2;
  for (int i = tid; i < job.count * quads; i += kAdThreads) {
    const int row = i / quads, at = row * a.inner_row + (i - row * quads) * 4;
    float4 s = *reinterpret_cast<const float4*>(part + at);
    for (int q = 1; q < deep; ++q) {
      const float4 v = *reinterpret_cast<const float4*>(part + q * 16 * a.inner_row + at);
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    *reinterpret_cast<float4*>(part + at) = s;
  }
  ad_cluster_arrive();
  const float scale = a.scale[job.slot];
  ad_cluster_wait();
  if (g0 < g1) {
    for (int i = tid; i < job.count * quads; i += kAdThreads) {
      const int row = i / quads, col = (i - row * quads) * 4;
      uint2 hi, lo;
      ad_split(ad_total<kC>(smem + (row * a.inner_row + col) * 4, scale), hi, lo);
      uint8_t* to = ad_smem + a.off_t + row * a.t_row + col * 2;
      *reinterpret_cast<uint2*>(to) = hi;
      *reinterpret_cast<uint2*>(to + a.rank * 2) = lo;
    }
  }
  ad_cluster_arrive();  // nobody reads another block's memory behind this
  __syncthreads();

  // ---- the second product: 32 columns at a time as four tiles of eight.  Tile j's column n is column 8 (n / 2) + 2 j + n % 2 of the 32, so that a lane has
  // eight columns side by side.  Lane t of a row's four has inner values 4t .. 4t + 3 of sixteen; where eight are left over, the two terms of
  // 2t and 2t + 1 share one step.
  const int full = a.rank >> 4;
  const bool tail = a.rank & 8;
  for (int g = g0 + warp, stage = 0; g < g1; g += kAdWarps, stage = stage + 1 == kStages ? 0 : stage + 1) {
    ad_wait<kStages - 1>();
    __syncwarp();
    const uint8_t* us = ad_smem + ring + stage * stage_bytes;
    const uint4 v0 = *reinterpret_cast<const uint4*>(us + 32 * a.u_row + lane * 16), v1 = *reinterpret_cast<const uint4*>(us + 32 * a.u_row + lane * 16 + 512);
    us += gid * a.u_row;
    const uint8_t* t0 = ad_smem + a.off_t + gid * a.t_row;
    const uint8_t* t1 = t0 + 8 * a.t_row;
    float o[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[j][i] = 0.f;
#pragma unroll
    for (int kb = 0; kb < kKB; ++kb) {
      if (kb < full) {
        const int at = 32 * kb + 8 * t;
        const uint2 h0 = *reinterpret_cast<const uint2*>(t0 + at), h1 = *reinterpret_cast<const uint2*>(t1 + at);
        const uint2 l0 = *reinterpret_cast<const uint2*>(t0 + a.rank * 2 + at), l1 = *reinterpret_cast<const uint2*>(t1 + a.rank * 2 + at);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint2 b = *reinterpret_cast<const uint2*>(us + 8 * j * a.u_row + at);
          ad_mma(o[j], h0.x, h1.x, h0.y, h1.y, b.x, b.y);
          ad_mma(o[j], l0.x, l1.x, l0.y, l1.y, b.x, b.y);
        }
      } else if (kb == full && tail) {
        const int at = 32 * kb + 4 * t;
        const uint32_t h0 = *reinterpret_cast<const uint32_t*>(t0 + at), h1 = *reinterpret_cast<const uint32_t*>(t1 + at);
        const uint32_t l0 = *reinterpret_cast<const uint32_t*>(t0 + a.rank * 2 + at), l1 = *reinterpret_cast<const uint32_t*>(t1 + a.rank * 2 + at);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t b = *reinterpret_cast<const uint32_t*>(us + 8 * j * a.u_row + at);
          ad_mma(o[j], h0, h1, l0, l1, b, b);
        }
      }
    }
    __syncwarp();
    fetch(g + kStages * kAdWarps, stage);
    const int col = job.begin + 32 * g + 8 * t, left = job.end - col;  // this lane's columns
    const bool whole = a.vec && left >= 8;
    const float f0[8] = {o[0][0], o[0][1], o[1][0], o[1][1], o[2][0], o[2][1], o[3][0], o[3][1]};
    const float f1[8] = {o[0][2], o[0][3], o[1][2], o[1][3], o[2][2], o[2][3], o[3][2], o[3][3]};
    uint16_t* out = (uint16_t*)a.out + col;
    if (row0 >= 0) ad_store(y + (long long)row0 * a.y_stride + col, out + (long long)row0 * a.out_stride, left, whole, v0, f0);
    if (row1 >= 0) ad_store(y + (long long)row1 * a.y_stride + col, out + (long long)row1 * a.out_stride, left, whole, v1, f1);
  }
  ad_cluster_wait();
}

// ---------------------------------------------------------------------------------------------------------------- portions: tcgen05
// Two launches.  First product: a cluster takes a tile of 128 rows (the M of tcgen05.mma) and all parts side by side (N), its blocks share the channels, 64
// at a time through a ring in shared memory; the sums go to a workspace as the second product's operand lies in shared memory.  Second product: a
// block takes a tile and a run of columns of a part, 128 at a time; K = the inner values' first terms and then their second ones.  With both in one
// launch, clusters of whole tiles were the unit that multiprocessors are filled by: 2000 rows of rank 64 beside [2048 -> 12288] took 55 us, of which the
// columns were 23, and in two 38.  The first one is bound by the latency of its chain, the second by memory.  What did not
// help there: y brought to L2 beside the first product (41 to 47 us), or no further than 2 or 4 column blocks ahead of the second (44 to 48).
// Operands lie in the 128-byte-swizzled K-major layout; they come by 16-byte asynchronous copies, since rows lie in any order and the columns of
// `up` are put so that the accumulator's fragments hold eight columns side by side.
// No block of a cluster may wait for tensor memory that another cluster's holds, as clusters could then wait for one another: ad_first sees to it that the
// blocks that fit a multiprocessor fit three quarters of its tensor memory, and the next kernel is not brought up before they have theirs.
__device__ __forceinline__ uint64_t ad_desc(uint32_t saddr) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(16u >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// kind::f16 instruction descriptor: fp32 accumulator, bf16 operands, both K-major, M = 128, N = n
__device__ __forceinline__ uint32_t ad_idesc(uint32_t n) { return (1u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((128u >> 4) << 24); }
__device__ __forceinline__ void ad_tc_mma(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"((uint32_t)add) : "memory");
}
__device__ __forceinline__ void ad_tc_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void ad_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void ad_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
// (of shared memory alone: one of all memory would wait for the stores to the result as well)
__device__ __forceinline__ void ad_proxy_fence() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }
// This thread's lane, eight columns.
__device__ __forceinline__ void ad_tc_ld8(uint32_t addr, float (&f)[8]) {
  uint32_t u[8];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\t"
      "tcgen05.wait::ld.sync.aligned;\n"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]) : "r"(addr) : "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(u[i]);
}
// Sixteen lanes, 32 columns, as the fragments of four tiles of 16 x 8: f[4 j + i], rows lane / 4 (i < 2) and lane / 4 + 8, columns 8 j + 2 (lane % 4) + i % 2.
__device__ __forceinline__ void ad_tc_ld_tiles(uint32_t addr, float (&f)[16]) {
  uint32_t u[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;\n"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]),
        "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
      : "r"(addr) : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(u[i]);
}

template <int kC, int kStages>
__global__ void __launch_bounds__(kAdThreads) adapter_first_kernel(const __grid_constant__ AdArgs a) {
  extern __shared__ uint8_t ad_raw[];
  __shared__ int rows_of[128];
  __shared__ __align__(8) uint64_t bars[kStages];
  __shared__ uint32_t tmem_word;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = (int)ad_cluster_rank();
  pdl_wait();
  // the parts that this cluster takes
  const int cl = blockIdx.x / kC, at = cl / a.part_groups, p0 = (cl - at * a.part_groups) * a.group_parts, np = min(a.group_parts, a.parts - p0);
  const int4 tile = __ldcg(a.tiles + at);
  const int row_of = tid < 128 ? ld_fresh(a.order + (long long)at * 128 + tid) : -1;  // (on its way beside the tile)
  const int count = tile.y;
  if (count <= 0 || tile.x < 0) return;  // (with the whole cluster)
  const uint32_t smem = ((uint32_t)__cvta_generic_to_shared(ad_raw) + 1023u) & ~1023u;
  uint8_t* base = ad_raw + (smem - (uint32_t)__cvta_generic_to_shared(ad_raw));
  const uint32_t bar = (uint32_t)__cvta_generic_to_shared(bars);
  if (tid < 128) rows_of[tid] = row_of;
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) dt_mbar_init(bar + 8 * s, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 0) {
    const uint32_t word = (uint32_t)__cvta_generic_to_shared(&tmem_word);
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(word), "r"(a.tmem_cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  ad_before_sync();
  __syncthreads();
  ad_after_sync();
  pdl_trigger();
  const uint32_t tmem = tmem_word;
  bool dead = false;

  const int inner = np * a.rank, inner16 = (inner + 15) & ~15, steps = (a.width + 63) >> 6;
  const uint16_t* down = (const uint16_t*)a.down + ((long long)tile.x * a.parts + p0) * a.rank * a.width;
  const int s0 = steps * rank / kC, n = steps * (rank + 1) / kC - s0;
  const uint32_t stage_bytes = 16384 + inner16 * 128;
  auto fetch = [&](int i) {
    if (i < n) {
      const uint32_t xs = smem + (i % kStages) * stage_bytes, ds = xs + 16384;
      const int k = 64 * (s0 + i) + 8 * (tid & 7);
      const bool in = k < a.width;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = (tid >> 3) + 32 * j, row = rows_of[r];
        const bool on = in && row >= 0;
        ad_copy16(xs + r * 128 + (((tid & 7) ^ (r & 7)) << 4), (const uint16_t*)a.x + (on ? (long long)row * a.x_stride + k : 0), on ? 16 : 0);
      }
      for (int r = tid >> 3; r < inner16; r += 32) {
        const bool on = in && r < inner;
        ad_copy16(ds + r * 128 + (((tid & 7) ^ (r & 7)) << 4), down + (on ? (long long)r * a.width + k : 0), on ? 16 : 0);
      }
    }
    ad_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages; ++i) fetch(i);
  for (int i = 0; i < n; ++i) {
    ad_wait<kStages - 2>();
    ad_proxy_fence();
    __syncthreads();
    if (tid == 0) {
      ad_after_sync();
      const uint32_t xs = smem + (i % kStages) * stage_bytes;
      const uint64_t da = ad_desc(xs), db = ad_desc(xs + 16384);
      const uint32_t idesc = ad_idesc(inner16);
#pragma unroll
      for (int j = 0; j < 4; ++j) ad_tc_mma(tmem, da + 2 * j, db + 2 * j, idesc, (i | j) != 0);
      ad_tc_commit(bar + 8 * (i % kStages));
    }
    if (i >= 1) {
      const int free = i - 1;  // its product has had a step's time
      if (free + kStages < n && !dt_mbar_wait(bar + 8 * (free % kStages), (free / kStages) & 1)) dead = true;
      fetch(free + kStages);
    }
  }
  if (n > 0 && !dt_mbar_wait(bar + 8 * ((n - 1) % kStages), ((n - 1) / kStages) & 1)) dead = true;
  ad_wait<0>();
  dead = __any_sync(0xffffffffu, dead);
  ad_after_sync();
  __syncthreads();  // (all copies into the ring have ended: the partial values lie over it)

  float* part = reinterpret_cast<float*>(base);
  const int q = warp & 3, half = warp >> 2;  // this warp's lanes of tensor memory; it shares them with another one
  if (32 * q < count) {
    for (int c = 8 * half; c < inner; c += 16) {
      float f[8];
      if (n > 0) {
        ad_tc_ld8(tmem + ((uint32_t)(32 * q) << 16) + c, f);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = 0.f;
      }
      float4* to = reinterpret_cast<float4*>(part + (32 * q + lane) * a.inner_row + c);
      to[0] = make_float4(f[0], f[1], f[2], f[3]);
      to[1] = make_float4(f[4], f[5], f[6], f[7]);
    }
  }
  ad_before_sync();
  ad_cluster_arrive();
  const float scale = a.scale[tile.x];
  ad_cluster_wait();
  // every block sums a share of the rows over all blocks
  const int quads = inner >> 2, rank16 = (a.rank + 15) & ~15, row0 = 128 / kC * rank;
  const int items = max(0, min(128 / kC, count - row0)) * quads;
  uint8_t* out = (uint8_t*)a.terms + ((long long)at * a.parts + p0) * a.blocks * 16384;
  constexpr int kMany = 8 / kC;  // of a thread's values on their way together
  for (int i0 = 0; i0 < items || i0 == 0; i0 += kMany * kAdThreads) {
    float4 sums[kMany];
#pragma unroll
    for (int m = 0; m < kMany; ++m) {
      const int i = i0 + m * kAdThreads + tid, r = i / quads;
      if (i < items) sums[m] = ad_total<kC>(smem + ((row0 + r) * a.inner_row + (i - r * quads) * 4) * 4, scale);
    }
    if (i0 + kMany * kAdThreads >= items) ad_cluster_arrive();  // (all of this block's reading is done)
#pragma unroll
    for (int m = 0; m < kMany; ++m) {
      const int i = i0 + m * kAdThreads + tid, r = i / quads, row = row0 + r, col = (i - r * quads) * 4, p = col / a.rank, j = col - p * a.rank;
      if (i >= items) break;
      uint2 hi, lo;
      ad_split(sums[m], hi, lo);
      uint8_t* to = out + (long long)p * a.blocks * 16384 + row * 128;
      const auto place = [&](int k) { return reinterpret_cast<uint2*>(to + (k >> 6) * 16384 + ((((k >> 3) & 7) ^ (row & 7)) << 4) + (k & 7) * 2); };
      *place(j) = hi;
      *place(rank16 + j) = lo;
      if (j >= a.rank - 8 && (a.rank & 8)) {  // what lies behind a term's values is zero
        *place(j + 8) = make_uint2(0, 0);
        *place(rank16 + j + 8) = make_uint2(0, 0);
      }
    }
  }
  asm volatile("fence.proxy.async.global;\n" ::: "memory");  // (the next kernel reads them by bulk copies)
  if (dead && a.status) atomicOr(a.status, B200KV_S_TIMEOUT);
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(a.tmem_cols) : "memory");
  ad_cluster_wait();  // nobody reads another block's memory behind this
}

// A block has a tile and a run of column blocks of one part; the runs of all tiles that have rows are as short as leaves them resident at once, or as long as
// a part.  How many tiles have rows only the plan knows, and most of its slots may be unused: 2000 rows of 4 adapters of rank 64 beside [2048 -> 12288] took
// 37.7, 62.7 and 102.3 us of 4, 64 and 256 slots with runs for as many tiles as there could be, and 37.0, 35.6 and 42.0 so.  Blocks behind the last run end at once.  Warps 0 to 7 add to y, a product's two halves of columns in four quarters of rows; one lane of
// warp 8 issues the products, into two accumulators in turn; warp 9 brings the columns of `up`, two blocks in shared memory or on their way.  Two blocks
// share a multiprocessor and hold half of its tensor memory each; neither waits for another one, so that a third could only wait for their end.
__global__ void __launch_bounds__(kAdSecondThreads, 2) adapter_second_kernel(const __grid_constant__ AdArgs a) {
  extern __shared__ uint8_t ad_raw[];
  __shared__ __align__(8) uint64_t bars[9];
  __shared__ uint32_t tmem_word;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, t = lane & 3;
  if (blockIdx.x == 0) pdl_wait();
  // What the first product's kernel waited for is in L2 as soon as this one is brought up, since every block of that one had its wait behind it then; but it is
  // not promised to this grid before its own wait, so L1, which may hold older lines, is passed by: the plan is read and y brought to L2.
  const int tiles = min(__ldcg(&a.tiles[0].z), a.max_tiles);
  const auto runs_of = [&](int part, int run) { return ((a.ends[part] - (part ? a.ends[part - 1] : 0) + kAdTcCols - 1) / kAdTcCols + run - 1) / run; };
  int blocks = 0, length = max(1, (a.col_blocks * tiles + a.room - 1) / a.room) - 1;  // (a tile's runs; of so many column blocks)
  do {
    ++length;
    blocks = 0;
    for (int p = 0; p < a.parts; ++p) blocks += runs_of(p, length);
  } while (blocks * tiles > a.room && blocks > a.parts);
  const int at_tile = blockIdx.x / blocks;
  if (at_tile >= tiles) return;  // (the first block has waited for the grid in front)
  int part = 0, run = blockIdx.x - at_tile * blocks;
  for (; part < a.parts - 1; ++part) {
    const int n = runs_of(part, length);
    if (run < n) break;
    run -= n;
  }
  const int begin = (part ? a.ends[part - 1] : 0) + run * length * kAdTcCols;
  const int cols = min(a.ends[part] - begin, length * kAdTcCols), products = (cols + kAdTcCols - 1) / kAdTcCols;
  const int4 tile = __ldcg(a.tiles + at_tile);
  const int32_t* order = a.order + (long long)at_tile * 128;
  const int q = warp & 3, half = (warp >> 2) & 1;  // this warp's lanes of tensor memory, its half of 128 columns
  const int lane_row = ld_fresh(order + 32 * q + lane);
  const int count = tile.y;
  if (count <= 0) return;
  if (tile.x < 0) {
    pdl_wait();
    if (a.out == a.y) return;
    if (warp < 8) ad_copy_rows<uint16_t>(a, ld_fresh(order + 16 * warp + (lane & 15)), count - 16 * warp, begin + lane, begin + cols, 32);
    return;
  }
  const uint32_t smem = ((uint32_t)__cvta_generic_to_shared(ad_raw) + 1023u) & ~1023u;
  const uint32_t bar = (uint32_t)__cvta_generic_to_shared(bars);
  const auto acc_full = [&](int i) { return bar + 8 * (i & 1); };
  const auto acc_free = [&](int i) { return bar + 16 + 8 * (i & 1); };
  const auto up_full = [&](int i) { return bar + 32 + 8 * (i & 1); };
  const auto up_free = [&](int i) { return bar + 48 + 8 * (i & 1); };
  const uint32_t bar_terms = bar + 64;
  // this lane's first column of its four rows
  int rows[4];
  const uint16_t* from[4];
  uint4 v[2][4] = {};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    rows[i] = __shfl_sync(0xffffffffu, lane_row, 8 * i + gid);
    from[i] = (const uint16_t*)a.y + (long long)max(rows[i], 0) * a.y_stride + begin + 64 * half + 8 * t;
  }
  auto load_y = [&](int c, int g) {  // 32 columns
    const bool whole = a.vec && cols - (kAdTcCols * c + 64 * half + 32 * g + 8 * t) >= 8;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (whole && rows[i] >= 0) v[g][i] = __ldcg(reinterpret_cast<const uint4*>(from[i] + kAdTcCols * c + 32 * g));
  };
  // y on its way to L2, so that no load waits for memory
  if (warp < 4 && a.vec && cols >= 8 && lane_row >= 0)
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;\n" ::"l"((const uint16_t*)a.y + (long long)lane_row * a.y_stride + begin), "r"(cols / 8 * 16) : "memory");
  const int rank16 = (a.rank + 15) & ~15, vecs = rank16 >> 3;
  const uint32_t us = smem + a.blocks * 16384, u_stage = ((rank16 + 63) >> 6) * kAdTcCols * 128;  // `up` lies behind the inner values
  auto fetch_up = [&](int c) {
    const uint16_t* up = (const uint16_t*)a.up + ((long long)tile.x * a.ends[a.parts - 1] + begin + kAdTcCols * c) * a.rank;
    const uint32_t dst = us + (c & 1) * u_stage;
    const unsigned by_vecs = (65536u + vecs - 1) / vecs;  // i / vecs of i < 512 by a product
    const long long next = 32ll * a.rank;
    const int left = cols - kAdTcCols * c;
#pragma unroll 2
    for (int i = lane; i < 32 * vecs; i += 32) {  // of each 32 columns
      const int at = (int)((unsigned)i * by_vecs >> 16), k = i - at * vecs;
      const int place = 8 * ((at >> 1) & 3) + 2 * (at >> 3) + (at & 1);
      const uint32_t to = dst + (k >> 3) * (kAdTcCols * 128) + place * 128 + (((k & 7) ^ (place & 7)) << 4);
      const int bytes = 8 * k < a.rank ? 16 : 0;
      const uint16_t* src = bytes ? up + at * a.rank + 8 * k : up;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const bool on = at + 32 * g < left;
        ad_copy16(to + g * 4096, on ? src : (const uint16_t*)a.up, on ? bytes : 0);
        src += next;
      }
    }
    ad_commit();
  };
  if (warp == 9) fetch_up(0);
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      dt_mbar_init(acc_full(i), 1);
      dt_mbar_init(acc_free(i), 8);
      dt_mbar_init(up_full(i), 1);
      dt_mbar_init(up_free(i), 1);
    }
    dt_mbar_init(bar_terms, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 8) {
    const uint32_t word = (uint32_t)__cvta_generic_to_shared(&tmem_word);
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(word), "r"(2 * kAdTcCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  ad_before_sync();
  __syncthreads();
  ad_after_sync();
  const uint32_t tmem = tmem_word;
  pdl_trigger();
  pdl_wait();
  bool dead = false;
  if (warp == 9) {
    for (int c = 1; c <= products; ++c) {
      if (c < products) {
        if (c >= 2 && !dt_mbar_wait(up_free(c), ((c >> 1) - 1) & 1)) dead = true;
        fetch_up(c);
        ad_wait<1>();
      } else {
        ad_wait<0>();
      }
      ad_proxy_fence();
      __syncwarp();
      if (lane == 0) dt_mbar_arrive(up_full(c - 1));
    }
  } else if (warp == 8) {
    if (lane == 0) {
      const uint32_t bytes = a.blocks * 16384;
      asm volatile("fence.proxy.async.global;\n" ::: "memory");
      dt_expect_tx(bar_terms, bytes);
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n"
                   ::"r"(smem), "l"((const uint8_t*)a.terms + ((long long)at_tile * a.parts + part) * bytes), "r"(bytes), "r"(bar_terms) : "memory");
      if (!dt_mbar_wait(bar_terms, 0)) dead = true;
      const uint32_t idesc = ad_idesc(kAdTcCols);
      const uint64_t da = ad_desc(smem), db = ad_desc(us);  // (in steps of 16 bytes)
      for (int c = 0; c < products; ++c) {
        if (!dt_mbar_wait(up_full(c), (c >> 1) & 1)) dead = true;
        if (c >= 2 && !dt_mbar_wait(acc_free(c), ((c >> 1) - 1) & 1)) dead = true;
        ad_after_sync();
        for (int k = 0; k < 2 * rank16; k += 16) {
          const int ku = k < rank16 ? k : k - rank16;
          ad_tc_mma(tmem + (c & 1) * kAdTcCols, da + (k >> 6) * 1024 + ((k & 63) >> 3),
                    db + (c & 1) * (u_stage >> 4) + (ku >> 6) * (kAdTcCols * 8) + ((ku & 63) >> 3), idesc, k != 0);
        }
        ad_tc_commit(acc_full(c));
        ad_tc_commit(up_free(c));
      }
    }
    __syncwarp();
  } else {
    load_y(0, 0);
    load_y(0, 1);
    for (int c = 0; c < products; ++c) {
      if (!dt_mbar_wait(acc_full(c), (c >> 1) & 1)) dead = true;
      dead = __any_sync(0xffffffffu, dead);
      ad_after_sync();
      if (32 * q < count && !dead) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const int at = kAdTcCols * c + 32 * g, left = cols - (at + 64 * half + 8 * t);
          const bool whole = a.vec && left >= 8;
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            float f[16];
            ad_tc_ld_tiles(tmem + ((uint32_t)(32 * q + 16 * m) << 16) + (c & 1) * kAdTcCols + 32 * g + 64 * half, f);
            const float f0[8] = {f[0], f[1], f[4], f[5], f[8], f[9], f[12], f[13]};
            const float f1[8] = {f[2], f[3], f[6], f[7], f[10], f[11], f[14], f[15]};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int i = 2 * m + h;
              uint16_t* to = (uint16_t*)a.out + (long long)rows[i] * a.out_stride + begin + 64 * half + 8 * t + at;
              if (rows[i] >= 0) ad_store(from[i] + at, to, left, whole, v[g][i], h ? f1 : f0);
            }
          }
          if (c + 1 < products) load_y(c + 1, g);
        }
      }
      ad_before_sync();
      __syncwarp();
      if (lane == 0) dt_mbar_arrive(acc_free(c));
    }
  }
  if (dead && a.status) atomicOr(a.status, B200KV_S_TIMEOUT);
  ad_before_sync();
  __syncthreads();
  if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(2 * kAdTcCols) : "memory");
}

// ---------------------------------------------------------------------------------------------------------------- CUDA cores
// 32-bit models, and bf16 rows that cannot be read in 16 bytes: sixteen rows a cluster, 32-bit products.  Bound by its chain of loads, so each thread has
// what it needs of sixteen rows on its way at once, y from the start: 40 rows of rank 8 beside [2048 -> 3456] 6.6 us, 13.6
// with a row's loads one after the other.
template <typename T>
__global__ void __launch_bounds__(kAdThreads) adapter_simt_kernel(const __grid_constant__ AdArgs a) {
  extern __shared__ __align__(16) uint8_t ad_smem[];
  __shared__ int rows_of[16];
  constexpr int kC = kAdSimtCluster;
  const uint32_t smem = (uint32_t)__cvta_generic_to_shared(ad_smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = (int)ad_cluster_rank();
  pdl_enter();
  pdl_wait();
  const AdJob job = ad_job<16, kC>(a);
  if (job.count <= 0) return;
  if (job.slot < 0) {
    if (a.out != a.y) ad_copy_rows<T>(a, ld_fresh(job.order + (lane & 15)), job.count, job.begin + rank * kAdThreads + tid, job.end, kC * kAdThreads);
    return;
  }
  const T* down = (const T*)a.down + ((long long)job.slot * a.parts + job.part) * a.rank * a.width;
  const T* up = (const T*)a.up + (long long)job.slot * a.ends[a.parts - 1] * a.rank;
  float* part = reinterpret_cast<float*>(ad_smem);
  float* xs = part + 16 * a.inner_row;
  if (tid < 16) rows_of[tid] = tid < job.count ? ld_fresh(job.order + tid) : -1;
  __syncthreads();
  // y of this thread's first column on its way
  const int cols = job.end - job.begin, c1 = job.begin + (int)((long long)cols * (rank + 1) / kC);
  int col = job.begin + (int)((long long)cols * rank / kC) + tid;
  float y[16];
  const auto load_y = [&]() {
#pragma unroll
    for (int r = 0; r < 16; ++r) y[r] = col < c1 && rows_of[r] >= 0 ? ld_fresh((const T*)a.y + (long long)rows_of[r] * a.y_stride + col) : 0.f;
  };
  load_y();
  const int k0 = (int)((long long)a.width * rank / kC), k1 = (int)((long long)a.width * (rank + 1) / kC);
  for (int i = tid; i < 16 * a.inner_row; i += kAdThreads) part[i] = 0.f;
  for (int s0 = k0; s0 < k1; s0 += kAdSimtChannels) {
    const int n = min(k1 - s0, kAdSimtChannels);
    float x[16], w[kAdSimtChannels / 32];
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = tid < n && rows_of[r] >= 0 ? ld_fresh((const T*)a.x + (long long)rows_of[r] * a.x_stride + s0 + tid) : 0.f;
    const auto load_w = [&](int j) {
#pragma unroll
      for (int i = 0; i < kAdSimtChannels / 32; ++i) w[i] = j < a.rank && lane + 32 * i < n ? ld_elem(down + (long long)j * a.width + s0 + lane + 32 * i) : 0.f;
    };
    load_w(warp);
    __syncthreads();  // (the channels before have been read)
#pragma unroll
    for (int r = 0; r < 16; ++r) xs[r * kAdSimtChannels + tid] = x[r];
    __syncthreads();
    for (int j = warp; j < a.rank; j += kAdWarps) {
      float s[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
      for (int i = 0; i < kAdSimtChannels / 32; ++i) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] += w[i] * xs[r * kAdSimtChannels + lane + 32 * i];
      }
      load_w(j + kAdWarps);
      // sums over the lanes: each step halves the rows that a lane has, so that in the end pairs of lanes have one
#pragma unroll
      for (int m = 8; m > 0; m >>= 1) {
        const bool high = lane & (2 * m);
#pragma unroll
        for (int r = 0; r < m; ++r) {
          const float other = __shfl_xor_sync(0xffffffffu, high ? s[r] : s[r + m], 2 * m);
          s[r] = (high ? s[r + m] : s[r]) + other;
        }
      }
      s[0] += __shfl_xor_sync(0xffffffffu, s[0], 1);
      if (!(lane & 1)) part[(lane >> 1) * a.inner_row + j] += s[0];
    }
  }
  ad_cluster_arrive();
  ad_cluster_wait();
  const int quads = a.rank >> 2;
  const float scale = a.scale[job.slot];
  for (int i = tid; i < 16 * quads; i += kAdThreads) {
    const int row = i / quads, col = (i - row * quads) * 4;
    *reinterpret_cast<float4*>(ad_smem + a.off_t + row * a.t_row + col * 4) = ad_total<kC>(smem + (row * a.inner_row + col) * 4, scale);
  }
  ad_cluster_arrive();
  __syncthreads();
  for (; col < c1; col += kAdThreads) {
    float d[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) d[r] = 0.f;
    const uint8_t* ts = ad_smem + a.off_t;
#pragma unroll 2
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
    for (int r = 0; r < 16; ++r)
      if (rows_of[r] >= 0) st_elem((T*)a.out + (long long)rows_of[r] * a.out_stride + col, y[r] + d[r]);
    if (col + kAdThreads < c1) {
      col += kAdThreads;
      load_y();
      col -= kAdThreads;
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
  cfg.numAttrs = take_early_launch(stream) ? 2 : 1;
  return launch_result(cudaLaunchKernelEx(&cfg, kernel, a));
}

// Shared memory of a block of few rows, and how it is laid out.
static size_t ad_rows_layout(AdArgs* a, int inner_blocks, int cluster, int stages, int most_cols) {
  a->inner_row = a->rank + 4;                    // (rows apart by other banks)
  a->t_row = (a->rank * 4 + 63) / 64 * 64 + 32;  // both terms; four rows at different banks
  a->u_row = a->rank * 2;
  while (a->u_row % 64 != 32) a->u_row += 16;    // four columns at different banks
  const int deep = a->rank <= 8 * inner_blocks ? kAdWarps : kAdWarps / 2;
  a->off_t = (uint32_t)(deep * 16 * a->inner_row * 4);
  a->off_u = a->off_t + 16 * a->t_row;
  a->ring = std::min(stages, ((most_cols + 31) / 32 + cluster * kAdWarps - 1) / (cluster * kAdWarps));  // (a warp has no more groups than that)
  return a->off_u + (size_t)kAdWarps * a->ring * (32 * a->u_row + 1024);
}

// The cluster for which rounds of clusters times a cluster's time are least.  By itself a cluster of C blocks takes about 3.6 us + (columns (21 + rank) + channels
// (13 + 0.3 rank)) 0.07 ns / C (rank 64 beside [2048 -> 12288] with 8, 4 and 2 blocks: 8.7, 13.5 and 22.2 us; rank 16 beside [2048 -> 2048] 4.3, 5.3 and 7.3).
// Blocks are resident by their shared memory (fewer at higher ranks beside wide parts) and registers; of the places for clusters of eight a seventh is left
// over, as a graphics cluster's multiprocessors are rarely a multiple of eight, but where three blocks share one.  us with 8, 4 and 2 blocks, 64 rows of 48
// adapters and then 16 of 16, the first taken up to rank 16 whatever the rank before (the last two of these 18.4 and 25.1 us):
//     rank 16: three parts of [2048 -> 4096] 15.1, 11.9, 8.6 and 6.5, 6.4, 7.4; two of [2048 -> 12288] 15.1, 12.5, 16.4 and 7.4, 8.1, 12.0; [6144 -> 2048] 7.6, 8.2, 10.2
//     rank 32: 18.2, 18.7, 20.9 and 7.4, 8.0, 9.5; 42.0, 30.1, 35.3 and 18.4, 10.5, 16.7; 10.1, 12.5, 19.4
//     rank 64: 31.2, 34.0, 27.5 and 12.5, 13.6, 12.3; 55.3, 41.4, 47.6 and 23.3, 13.8, 22.7; 19.2, 26.3, 24.3
template <int kNT, int kKB, int kStages>
static int ad_rows(const AdArgs& args, int clusters, int tiles, int most_cols, cudaStream_t stream) {
  constexpr int kShared = 228 * 1024;  // of a multiprocessor; a block has one of these KB to itself
  const int sms = device_sms(), used = tiles * args.parts;
  const long long work = (long long)most_cols * (21 + args.rank) + (long long)args.width * (13 + 3 * args.rank / 10);
  AdArgs a = args, best = args;
  long long least = 0;
  int cluster = 0;
  size_t smem = 0;
  for (int c = 8; c >= 2; c /= 2) {
    const size_t bytes = ad_rows_layout(&a, kNT, c, kStages, most_cols);
    const int fit = std::min(ad_rows_blocks(kKB), (int)(kShared / (bytes + 1024))), room = c == 8 && fit < 3 ? sms * fit * 6 / 7 : sms * fit;
    const long long cost = ((long long)used * c + room - 1) / std::max(room, 1) * (50000 + work / c);
    if (cluster && cost >= least) continue;
    least = cost;
    cluster = c;
    smem = bytes;
    best = a;
  }
  if (cluster == 8) return ad_launch(adapter_rows_kernel<kNT, kKB, 8, kStages>, best, clusters, 8, smem, stream);
  if (cluster == 4) return ad_launch(adapter_rows_kernel<kNT, kKB, 4, kStages>, best, clusters, 4, smem, stream);
  return ad_launch(adapter_rows_kernel<kNT, kKB, 2, kStages>, best, clusters, 2, smem, stream);
}

// Tiles of 128 rows: the parts of a cluster, tensor memory and shared memory of the first product.
static size_t ad_first(AdArgs* a, int stages) {
  a->group_parts = a->parts * a->rank <= 256 ? a->parts : 256 / a->rank;
  a->part_groups = (a->parts + a->group_parts - 1) / a->group_parts;
  const int inner = a->group_parts * a->rank, inner16 = (inner + 15) / 16 * 16;
  a->tmem_cols = 32;
  while ((int)a->tmem_cols < inner16) a->tmem_cols *= 2;
  a->inner_row = inner + 4;  // (rows apart by other banks)
  const size_t ring = (size_t)stages * (16384 + inner16 * 128), partial = (size_t)128 * a->inner_row * 4;
  const size_t all = 1024 + (ring > partial ? ring : partial), least = (a->tmem_cols > 128 ? 116 : 60) * 1024;  // one block a multiprocessor, three
  return all > least ? all : least;
}
static int ad_terms_blocks(int rank) { return (2 * ((rank + 15) / 16 * 16) + 63) / 64; }

}  // namespace b200kv

using namespace b200kv;

static int ad_check_plan(const b200dec_adapter_plan_t* plan) {
  if (!plan->order || !plan->tiles) return B200KV_E_NULL;
  if (plan->num_rows < 0 || plan->num_rows > (1 << 24) || plan->slots < 1 || plan->slots > kAdMaxSlots) return B200KV_E_RANGE;
  if (plan->tile_rows != 16 && plan->tile_rows != 128) return B200KV_E_SHAPE;
  if (plan->max_tiles < plan->num_rows / plan->tile_rows + (plan->num_rows < plan->slots + 1 ? plan->num_rows : plan->slots + 1)) return B200KV_E_WORKSPACE;
  if ((long long)plan->max_tiles * plan->tile_rows * kAdMaxParts > 0x0fffffffLL || (plan->tile_rows == 128 && plan->max_tiles > 65535)) return B200KV_E_RANGE;
  return aligned(plan->tiles, 16) && aligned(plan->order, 4) ? B200KV_OK : B200KV_E_ALIGN;
}

extern "C" int b200dec_adapter_plan(const int32_t* ids, const b200dec_adapter_plan_t* plan, int32_t* status, void* stream) {
  if (!plan) return B200KV_E_NULL;
  if (plan->num_rows == 0) return B200KV_OK;
  if (!ids) return B200KV_E_NULL;
  if (int rc = ad_check_plan(plan)) return rc;
  if (!aligned(ids, 4)) return B200KV_E_ALIGN;
  // us with 256, 512 and 1024 threads, a row fetched at a time: 64 rows of 48 adapters 3.4, 3.7 and 4.6, 1000 rows 6.7, 6.2 and 7.3, 2000 rows 10.4, 9.1 and 9.8
  const int threads = plan->num_rows <= 256 && plan->slots < 256 ? kAdPlanThreads / 2 : kAdPlanThreads;
  return launch_result(launch_kernel(take_early_launch((cudaStream_t)stream), adapter_plan_kernel, dim3(1), dim3(threads), (size_t)(plan->slots + 1) * 4, (cudaStream_t)stream, ids, (int)plan->num_rows,
                                      (int)plan->slots, (int)plan->tile_rows, plan->order, (int4*)plan->tiles, (int)plan->max_tiles, status));
}

// Clusters of sixteen rows and a part that can have any.
static long long ad_used(const b200dec_adapters* ad, const b200dec_adapter_plan_t* plan) {
  const long long tiles = plan->num_rows / 16 + std::min(plan->num_rows, plan->slots + 1);
  return ad->parts * std::min(tiles, (long long)plan->max_tiles * (plan->tile_rows / 16));
}

// Whether tiles of 128 rows go to tcgen05 in whole, and not sixteen rows by sixteen to mma.sync, as a plan of small tiles does.  The latter is one launch
// without a workspace, and a row's weights are little at a low rank; at a higher one every sixteen rows fetch them again.  us, mma.sync and
// tcgen05, four adapters:
//     rank 16, three parts of [2048 -> 4096]: 1000 rows (201 clusters) 12.2 and 14.8, 1250 rows (249) 18.4 and 15.2
//     rank 16, two parts of [2048 -> 12288]: 1500 rows (196) 24.3 and 27.1, 1750 rows (228) 32.9 and 28.8
//     rank 32, [2048 -> 2048]: 1000 rows (67) 9.4 and 12.0, 1250 rows (83) 15.8 and 12.2; two parts of [2048 -> 12288]: 300 rows (46) 23.7 and 15.7
//     rank 64, [2048 -> 2048]: 512 rows (37) 18.0 and 11.5
static bool ad_whole_tiles(const b200dec_adapters* ad, const b200dec_adapter_plan_t* plan) {
  if (plan->tile_rows != 128) return false;
  int most = 0;
  for (int p = 0; p < ad->parts && p < kAdMaxParts; ++p) most = std::max(most, ad->ends[p] - (p ? ad->ends[p - 1] : 0));
  const long long used = ad_used(ad, plan);
  return ad->rank <= 16 ? 2 * used > 3 * device_sms() : ad->rank > 32 || most > 4096 || 2 * used > device_sms();
}

extern "C" size_t b200dec_add_adapters_workspace(const b200dec_adapters* ad, const b200dec_adapter_plan_t* plan) {
  if (!ad || !plan || !ad_whole_tiles(ad, plan) || ad->elem != 2 || plan->max_tiles < 1 || ad->parts < 1 || ad->rank < 8) return 0;
  return (size_t)plan->max_tiles * ad->parts * ad_terms_blocks(ad->rank) * 16384;
}

extern "C" int b200dec_add_adapters(const b200dec_adapters* ad, const b200dec_adapter_plan_t* plan, const void* x, int64_t x_stride, const void* y,
                                    int64_t y_stride, void* out, int64_t out_stride, void* workspace, size_t workspace_bytes, int32_t* status,
                                    void* stream) {
  if (!ad || !plan) return B200KV_E_NULL;
  if (plan->num_rows == 0) return B200KV_OK;
  if (!ad->down || !ad->up || !ad->scale || !x || !y || !out) return B200KV_E_NULL;
  if (int rc = ad_check_plan(plan)) return rc;
  if (ad->slots != plan->slots) return B200KV_E_SHAPE;
  if (ad->elem != 2 && ad->elem != 4) return B200KV_E_SHAPE;
  if (ad->parts < 1 || ad->parts > kAdMaxParts || ad->rank < 8 || ad->rank > 128 || ad->rank % 8 || ad->width < 1) return B200KV_E_SHAPE;
  if (ad->width > (1 << 24)) return B200KV_E_RANGE;
  const int max_tiles = plan->max_tiles, tile_rows = plan->tile_rows;
  const int32_t *order = plan->order, *tiles = plan->tiles;
  AdArgs a = {};
  a.down = ad->down; a.up = ad->up; a.scale = ad->scale; a.x = x; a.y = y; a.out = out;
  a.x_stride = x_stride; a.y_stride = y_stride; a.out_stride = out_stride;
  a.order = order; a.tiles = (const int4*)tiles; a.tile_rows = tile_rows; a.max_tiles = max_tiles;
  a.rank = ad->rank; a.width = ad->width; a.parts = ad->parts; a.status = status;
  bool even = true;
  int most = 0;
  for (int p = 0, begin = 0; p < ad->parts; ++p) {
    if (ad->ends[p] <= begin || ad->ends[p] > (1 << 24)) return B200KV_E_SHAPE;
    even = even && begin % 8 == 0;
    a.ends[p] = ad->ends[p];
    if (ad->ends[p] - begin > most) most = ad->ends[p] - begin;
    begin = ad->ends[p];
  }
  const int cols = a.ends[a.parts - 1];
  if (x_stride < a.width || y_stride < cols || out_stride < cols || out == x) return B200KV_E_SHAPE;
  if (out == y && out_stride != y_stride) return B200KV_E_SHAPE;
  if (!aligned(ad->down, 16) || !aligned(ad->up, 16) || !aligned(ad->scale, 4) || !aligned(x, ad->elem) || !aligned(y, ad->elem) || !aligned(out, ad->elem))
    return B200KV_E_ALIGN;
  a.vec = even && aligned(y, 16) && aligned(out, 16) && y_stride % 8 == 0 && out_stride % 8 == 0;
  cudaStream_t s = (cudaStream_t)stream;
  const int clusters = max_tiles * a.parts, fine = clusters * (tile_rows / 16);  // the latter with sixteen rows each
  if (ad->elem == 4 || a.width % 8 || x_stride % 8 || !aligned(x, 16)) {
    a.inner_row = a.rank;
    a.t_row = a.rank * 4;
    a.off_t = 16u * a.inner_row * 4 + 16u * kAdSimtChannels * 4;
    const size_t smem = a.off_t + (size_t)16 * a.t_row;
    return ad->elem == 4 ? ad_launch(adapter_simt_kernel<float>, a, fine, kAdSimtCluster, smem, s)
                         : ad_launch(adapter_simt_kernel<uint16_t>, a, fine, kAdSimtCluster, smem, s);
  }
  if (ad_whole_tiles(ad, plan)) {
    a.blocks = ad_terms_blocks(a.rank);
    a.terms = workspace;
    if (!workspace || workspace_bytes < b200dec_add_adapters_workspace(ad, plan)) return B200KV_E_WORKSPACE;
    if (!aligned(workspace, 16)) return B200KV_E_ALIGN;
    // Clusters are of eight blocks where that many fit at once (a graphics cluster's multiprocessors are rarely a multiple of eight: about a seventh is left
    // over), else of four, and copies run as far ahead as leaves room for as many blocks.  us of both products with 8 blocks and 3, 4 or 5 stages, and with 4
    // and 5: 1000 rows of rank 64 (12 clusters) beside [2048 -> 2048] 13.8, 13.5, 12.4, 14.8, beside [6144 -> 2048] 19.2, 18.4, 17.1, 24.5; 2000 rows of rank
    // 64 (19) beside these 18.6, 17.1, 20.9, 17.0 and 24.6, 22.7, 30.6, 26.9, beside three parts of [2048 -> 4096] (one block a multiprocessor) 31.4, 29.4,
    // 29.5, 24.3; of rank 16 beside [2048 -> 12288] 33.3, 32.8, 40.3, 42.1.  Where the columns are most of the work, few blocks that leave room for none of the
    // second product's beside them are the faster at higher ranks: beside [2048 -> 12288], 2000 rows of rank 64 44.0, 40.1, 40.2, 37.3, 4000 of rank 32 79.0,
    // 85.0, 67.5, 63.0.
    const size_t smem = ad_first(&a, 3), more = ad_first(&a, 4), deep = ad_first(&a, 5);
    const int first = max_tiles * a.part_groups, sms = device_sms(), room = sms * 6 / 7;
    // clusters that are likely to have rows: an adapter's last tile is half full
    const int groups = std::min(plan->num_rows, plan->slots + 1), used = a.part_groups * (int)std::min<long long>(max_tiles, (plan->num_rows + 64ll * groups + 127) / 128);
    const auto fits = [&](size_t bytes) { return used * 8 <= room * (int)(227 * 1024 / (bytes + 2048)); };
    int rc;
    if (used * 8 > room && deep <= kAdMostSmem && a.rank > 16 && cols >= 4 * a.width) rc = ad_launch(adapter_first_kernel<4, 5>, a, first, 4, deep, s);
    else if (used * 8 <= room && deep <= kAdMostSmem) rc = ad_launch(adapter_first_kernel<8, 5>, a, first, 8, deep, s);
    else if (fits(more)) rc = ad_launch(adapter_first_kernel<8, 4>, a, first, 8, more, s);
    else if (fits(smem)) rc = ad_launch(adapter_first_kernel<8, 3>, a, first, 8, smem, s);
    else if (used * 4 <= room && deep <= kAdMostSmem) rc = ad_launch(adapter_first_kernel<4, 5>, a, first, 4, deep, s);
    else rc = ad_launch(adapter_first_kernel<4, 3>, a, first, 4, smem, s);
    if (rc) return rc;
    const int ublocks = ((a.rank + 15) / 16 * 16 + 63) / 64;
    a.room = 2 * sms;
    for (int p = 0, begin = 0; p < a.parts; begin = a.ends[p++]) a.col_blocks += (a.ends[p] - begin + kAdTcCols - 1) / kAdTcCols;
    // as many blocks as any number of tiles can have runs.  2000 rows of rank 64 beside [2048 -> 12288], all on clusters of eight: 42 us with runs for one
    // round of blocks, 48 with runs of a single column block, 47 with runs one longer, 54 with three longer
    const dim3 grid((unsigned)std::min((long long)max_tiles * a.col_blocks, std::max<long long>(a.room, (long long)max_tiles * a.parts)));
    const size_t second = 1024 + (size_t)a.blocks * 16384 + (size_t)2 * ublocks * kAdTcCols * 128;
    auto kernel = adapter_second_kernel;
    if (!allow_smem(kernel, kAdMostSmem)) return launch_result(cudaErrorInvalidValue);
    // brought up while the first one runs, also in recorded steps: it waits for it, and nothing else stands between them
    return launch_result(launch_kernel(b200kv_get_early_launch() != 0, kernel, grid, dim3(kAdSecondThreads), second, s, a));
  }
  const int kb = (a.rank + 15) / 16;
  // tiles of sixteen rows that can be expected: every slot in use, and by as many rows (what is in use only the device knows)
  const int groups = std::min(plan->num_rows, plan->slots + 1), used = std::min(fine / a.parts, groups * ((plan->num_rows + 16 * groups - 1) / (16 * groups)));
  if (kb <= 1) return ad_rows<2, 1, 3>(a, fine, used, most, s);
  if (kb <= 2) return ad_rows<4, 2, 3>(a, fine, used, most, s);
  if (kb <= 4) return ad_rows<8, 4, 2>(a, fine, used, most, s);
  return ad_rows<8, 8, 2>(a, fine, used, most, s);
}
