// What every request asks of its next token: penalties for repeated tokens, biases and grammar masks on its logits, and the choice with
// its own temperature, top-k, top-p and min-p.  (The sampler of sampler.cu has one temperature for all rows and nothing on the logits.)
//
// Adjusted logit of token v, in 32 bits, each operation rounded by itself:
//     l = l > 0 ? l / repetition : l * repetition     if v stands in the history (prompt or output)
//     l = l - (frequency * n + presence)              if v stands n > 0 times in the output
//     l = l + the sum of its biases, in their order
//     l = -inf                                        if the mask has no bit for it
// How often a token was said is counted in shared memory, by each block for its own columns: a history is short beside a vocabulary, so every
// block reads all of it, from L2.
//
// The choice: one cluster of blocks holds a row's adjusted logits in shared memory, so the logits are read once and everything behind that
// happens on the multiprocessors.  With m the largest, z = (m - l) / temperature and w = exp(-z), tokens are ordered by l (equal ones by
// index).  Kept are the first top_k; of these the shortest run whose weight is at least top_p of theirs; of these the ones with w >= min_p.
// The token is the first, by index, at which the kept weights so far exceed uniform * their sum.
//
// Few tokens are kept, mostly.  A thread's largest logit is a token, so as many tokens are above a floor as threads' largest are: a histogram of those alone,
// one addition a thread, gives a floor with at least k tokens above it and few more (64 of 151936: 64 to 83, 200: 202 to 400), where one of all tokens cost
// an addition for each in reach.  One block takes the tokens above the floor from the others, which end, puts them in order and draws.  Where they are too many, or
// the share of weight lies further out, a cut is found by a histogram of z (counts, and weights as integers, so that no order of additions matters) over the
// likelier tokens, or over the others if it does not lie there, down to the few tokens of one bin, which are sorted.  Bins are of z, or of what z would be at
// a temperature of 64 where that is higher (else tokens in order would share one); where they do not reach a cut, or too many tokens share the
// smallest, they are of the logits' own bits, ten at a time.  Blocks tell one another sums of bins, and
// read from one another only the bins among which the cut lies.  A token of top-k of 64 requests took 42 us that way, and 25 by a floor.
//
// Precision: 32-bit logits and weights (two steps of the last place from the exponential), sums of them in 32 bits within a warp and in 64 beyond; a weight's
// integer is in steps of 2^-32 of the largest one, sums of those are in 64 bits.
//
// Measured: rules for 64 rows of 151936 bf16 logits and histories of up to 8192 tokens 22 us (58 MB, 2.6 TB/s), for a row of 32768 4.3.  Choice for 64 such
// rows with settings of their own 54 us, without cuts 33, for one row 15.  What bounds both is not the bytes but chains: entry, history, row,
// largest logit, weights, floor, list, draw, each a few hundred cycles of memory or a barrier of the cluster (1 to 1.5 us each beside another block), and that
// in two rounds of blocks for a full batch, whose rows of 32 bits (39 MB) do not fit the multiprocessors' memory (33 MB) at once.
#include "dec_common.cuh"

namespace b200kv {

struct TcRules {
  int32_t* history;
  const int32_t *slots, *lengths, *prompts;
  const float *repetition, *presence, *frequency;
  const int32_t* bias_ids;
  const float* bias;
  const uint32_t* masks;
  const int32_t* mask_rows;
  int capacity, num_histories, num_bias, num_masks, mask_words;
};

// What the rules are for one entry.
struct TcEntry {
  bool idle;
  int slot, length, prompt;
  float repetition, presence, frequency;
  bool penalties;
  const int32_t* history;
  const uint32_t* mask;  // NULL: everything is allowed
};

__device__ __forceinline__ TcEntry tc_entry(const TcRules& r, int e, bool report, int32_t* status) {
  TcEntry t;
  // (all on their way before the first is looked at)
  t.slot = r.slots ? r.slots[e] : e;
  t.length = r.history ? r.lengths[e] : 0;
  t.prompt = r.history && r.prompts ? r.prompts[e] : 0x7fffffff;
  t.repetition = r.repetition ? r.repetition[e] : 1.f;
  t.presence = r.presence ? r.presence[e] : 0.f;
  t.frequency = r.frequency ? r.frequency[e] : 0.f;
  const int m = r.masks ? r.mask_rows[e] : -1;
  bool bad = false;
  t.idle = t.slot < 0;
  if (t.slot < -1 || (r.history && t.slot >= r.num_histories)) { bad = true; t.idle = true; }
  t.history = nullptr;
  if (t.idle || !r.history) {
    t.length = 0;
  } else {
    if (t.length < 0 || t.length > r.capacity || t.prompt < 0) bad = true;
    if (t.length >= 0) t.history = r.history + (long long)t.slot * r.capacity;  // (nothing is appended behind a length that is none)
    t.length = max(0, min(t.length, r.capacity));
  }
  t.penalties = t.length > 0 && (t.repetition != 1.f || t.presence != 0.f || t.frequency != 0.f);
  t.mask = nullptr;
  if (m >= 0 && m < r.num_masks) t.mask = r.masks + (long long)m * r.mask_words;
  else if (m != -1) bad = true;
  if (bad && report && status) atomicOr(status, B200KV_S_BAD_POSITION);
  return t;
}

constexpr uint32_t kTcSeen = 0x80000000u;  // in the prompt, beside how often a token stands in the output

// table[v - v0] for the columns v0 .. v0 + n of this block; cleared by the caller, with a barrier on both sides.  A thread takes four tokens at a
// time, and fetches those of four times together.
__device__ __forceinline__ void tc_count(const TcEntry& t, int V, int v0, int n, uint32_t* table, bool report, int32_t* status) {
  auto take = [&](int i, int id) {
    const int at = id - v0;
    if ((unsigned)at < (unsigned)n) {
      if (i >= t.prompt) atomicAdd(&table[at], 1u);
      else if (!(*(volatile uint32_t*)&table[at] & kTcSeen)) atomicOr(&table[at], kTcSeen);
    }
    if (report && (unsigned)id >= (unsigned)V && status) atomicOr(status, B200KV_S_BAD_POSITION);
  };
  const int head = min(t.length, (int)((16 - (reinterpret_cast<uintptr_t>(t.history) & 15)) & 15) / 4), quads = (t.length - head) / 4;
  const int4* p = reinterpret_cast<const int4*>(t.history + head);
  for (int i = threadIdx.x; i < quads; i += 4 * blockDim.x) {
    int4 q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j * (int)blockDim.x < quads) q[j] = __ldcg(p + i + j * blockDim.x);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = head + 4 * (i + j * (int)blockDim.x);
      if (i + j * (int)blockDim.x < quads) {
        take(at, q[j].x);
        take(at + 1, q[j].y);
        take(at + 2, q[j].z);
        take(at + 3, q[j].w);
      }
    }
  }
  // in front of the first sixteen bytes, and behind the last
  const int rest = t.length - 4 * quads;
  if ((int)threadIdx.x < rest) {
    const int i = (int)threadIdx.x < head ? threadIdx.x : 4 * quads + threadIdx.x;
    take(i, __ldcg(t.history + i));
  }
}

__device__ __forceinline__ float tc_penalised(const TcEntry& t, float l, uint32_t seen) {
  if (seen) {
    l = l > 0.f ? __fdiv_rn(l, t.repetition) : __fmul_rn(l, t.repetition);
    const uint32_t n = seen & ~kTcSeen;
    if (n) l = __fsub_rn(l, __fadd_rn(__fmul_rn(t.frequency, (float)n), t.presence));
  }
  return l;
}
__device__ __forceinline__ bool tc_allowed(const TcEntry& t, int v) { return !t.mask || (t.mask[v >> 5] >> (v & 31) & 1u); }

// The biases of this block's columns on values that the block holds: every token's own, in order, by the thread of its first one.
template <typename Add>
__device__ __forceinline__ void tc_bias(const TcRules& r, const TcEntry& t, int e, int V, int v0, int n, bool report, int32_t* status, Add add) {
  const int32_t* ids = r.bias_ids + (long long)e * r.num_bias;
  const float* bias = r.bias + (long long)e * r.num_bias;
  for (int i = threadIdx.x; i < r.num_bias; i += blockDim.x) {
    const int id = ids[i];
    if (report && (id < -1 || id >= V) && status) atomicOr(status, B200KV_S_BAD_POSITION);
    if (id < v0 || id >= v0 + n || !tc_allowed(t, id)) continue;
    bool first = true;
    for (int j = 0; j < i && first; ++j) first = ids[j] != id;
    if (!first) continue;
    float s = bias[i];
    for (int j = i + 1; j < r.num_bias; ++j)
      if (ids[j] == id) s = __fadd_rn(s, bias[j]);
    add(id, s);
  }
}

// Four logits as they come from memory, so that several can be on their way.  (Four, so that a warp writes whole lines of 32-bit values.)  Through L2, as the
// histories: the kernel in front may have written them, rules on logits for one, beside which this one is brought up.
// (Rows that are not aligned to four logits go one by one: rules for 64 rows of 151937 bf16 logits 36 us, for 151936 22; choices 53 and 54.)
template <typename T>
struct TcRaw;
template <>
struct TcRaw<uint16_t> {
  uint2 a;
  __device__ __forceinline__ void load(const uint16_t* p) { a = __ldcg(reinterpret_cast<const uint2*>(p)); }
  __device__ __forceinline__ void get(float (&f)[4]) const {
    f[0] = __uint_as_float(a.x << 16); f[1] = __uint_as_float(a.x & 0xFFFF0000u);
    f[2] = __uint_as_float(a.y << 16); f[3] = __uint_as_float(a.y & 0xFFFF0000u);
  }
};
template <>
struct TcRaw<float> {
  float4 a;
  __device__ __forceinline__ void load(const float* p) { a = __ldcg(reinterpret_cast<const float4*>(p)); }
  __device__ __forceinline__ void get(float (&f)[4]) const { f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; }
};
// Penalties and mask on four logits from column v on (a multiple of four).
__device__ __forceinline__ void tc_settle(const TcEntry& t, int v, const uint32_t* seen, float (&f)[4]) {
  if (t.penalties) {
    const uint4 n = *reinterpret_cast<const uint4*>(seen);
    if (n.x | n.y | n.z | n.w) {  // (few are)
      f[0] = tc_penalised(t, f[0], n.x);
      f[1] = tc_penalised(t, f[1], n.y);
      f[2] = tc_penalised(t, f[2], n.z);
      f[3] = tc_penalised(t, f[3], n.w);
    }
  }
  if (!t.mask) return;
  const uint32_t bits = t.mask[v >> 5] >> (v & 31);
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = bits >> j & 1u ? f[j] : -INFINITY;
}

// ---------------------------------------------------------------------------------------------------------------- adjusted logits
constexpr int kAjThreads = 512;
constexpr int kAjCols = kAjThreads * 4;  // of a block, times kAhead

// grid (column blocks, entries).  kAhead: times that a thread takes four columns.  vec: rows aligned to four elements on both sides.  The logits are on
// their way while the history is counted; the few that have a bias change where they lie.  (Reading back and changing only the columns that the history
// names, beside a plain copy, took 26 to 30 us for 64 rows of 151936, a table for all columns 22.)  The registers of two blocks a multiprocessor: with those
// that eight times four 32-bit logits ask for there was one, and 64 rows of 151936 took 34.8 us instead of 25.2.
template <typename T, int kAhead>
__global__ void __launch_bounds__(kAjThreads, kAhead > 2 || sizeof(T) == 4 ? 2 : 3)
adjust_logits_kernel(const T* logits, long long stride, const TcRules r, float* out, long long out_stride, int V, bool vec, int32_t* status) {
  extern __shared__ __align__(16) uint32_t aj_table[];
  uint32_t* table = aj_table;
  pdl_enter();
  pdl_wait();
  const int e = blockIdx.y, v0 = blockIdx.x * (kAhead * kAjCols), n = min(kAhead * kAjCols, V - v0), tid = threadIdx.x;
  const bool report = blockIdx.x == 0;
  const T* src = logits + (long long)e * stride + v0;
  float* dst = out + (long long)e * out_stride + v0;
  TcRaw<T> ahead[kAhead];
#pragma unroll
  for (int s = 0; s < kAhead; ++s) {
    const int i = 4 * (tid + s * kAjThreads);
    if (vec && i + 4 <= n) ahead[s].load(src + i);
  }
  for (int i = 4 * tid; i < kAhead * kAjCols; i += 4 * kAjThreads) *reinterpret_cast<uint4*>(table + i) = make_uint4(0, 0, 0, 0);
  const TcEntry t = tc_entry(r, e, report && tid == 0, status);
  if (t.idle) return;
  if (t.penalties) {
    __syncthreads();
    tc_count(t, V, v0, n, table, report, status);
    __syncthreads();
  }
#pragma unroll
  for (int s = 0; s < kAhead; ++s) {
    const int i = 4 * (tid + s * kAjThreads);
    if (i >= n) break;
    float f[4];
    const bool whole = vec && i + 4 <= n;
    if (whole) {
      ahead[s].get(f);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = i + j < n ? ld_fresh(src + i + j) : 0.f;
    }
    tc_settle(t, v0 + i, table + i, f);
    if (whole) {
      st_vec(dst + i, f);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + j < n) dst[i + j] = f[j];
    }
  }
  if (r.num_bias) {
    __syncthreads();  // what the block's other threads wrote
    tc_bias(r, t, e, V, v0, n, report, status, [&](int id, float s) { dst[id - v0] = __fadd_rn(ld_fresh(dst + id - v0), s); });
  }
}

// ---------------------------------------------------------------------------------------------------------------- the choice
constexpr int kTcThreads = 512;
constexpr int kTcWarps = kTcThreads / 32;
constexpr int kTcMaxCluster = 8;
constexpr int kTcBins = 1024, kTcCoarse = 32;  // and sums of 32 bins
constexpr int kTcMembers = 1024;               // tokens of one bin that are put in order
constexpr int kTcMaxLocal = 48 * 1024;         // columns of a block
constexpr int kTcShort = 512;                  // likely tokens that are drawn from without histograms of all: one a thread
constexpr int kTcShare = 112;                  // of them that are looked for where a share of the weight is kept: of 300 rows of 151936 and shares of
                                               // 0.5 to 0.99, 282 need 44 tokens at most, the others thousands
constexpr int kTcPlaces = 256;                 // of the threads' largest logits: 32 an octave of z + 0.5, up to a z of 127.5
constexpr uint32_t kTcNoPlace = 1u << 20;
constexpr int kTcShortWarp = 64;               // of a warp's columns
static_assert(kTcShort == kTcThreads && kTcShortWarp * kTcWarps <= kTcMembers && 2 * kTcMembers + 2 * kTcPlaces <= 3 * kTcBins &&
              kTcMembers == 2 * kTcThreads, "places of the likely tokens");
constexpr uint32_t kTcRowAt = kTcBins * 12 + kTcMembers * 8;  // the histogram, a bin's tokens, the row

struct TcDraw {
  const float* temperature;
  const int32_t* top_k;
  const float *top_p, *min_p, *uniform;
};

// What the blocks of a cluster tell one another; every block has a copy of its own.
struct TcMail {
  float best[kTcMaxCluster];
  float rest[kTcMaxCluster];
  int first[kTcMaxCluster], equal[kTcMaxCluster];  // of the largest ones
  double mass[kTcMaxCluster];    // the weights that are drawn from
  float weight[kTcMaxCluster];   // of the tokens among which a share is kept
  uint32_t coarse[2][kTcCoarse];   // of this block: sums of 32 bins
  uint32_t listed_by[kTcMaxCluster];
  uint32_t likely[kTcMaxCluster];  // number of likely tokens; kTcNoPlace: some warp had no place for its own
  unsigned long long listed_mass[kTcMaxCluster];  // the likely tokens' weights
  uint32_t ties[kTcMaxCluster];
  // within the block
  uint32_t fetched[2][kTcMaxCluster][kTcCoarse];
  uint32_t listed;
  unsigned long long some_mass;  // of the first k
  unsigned long long cut;  // a token's key
  int cut_at;
};

__device__ __forceinline__ int tc_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return (int)r;
}
__device__ __forceinline__ int tc_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return (int)r;
}
__device__ __forceinline__ void tc_cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// The address of a variable of this block in block `rank`'s shared memory.
__device__ __forceinline__ uint32_t tc_there(const void* p, int rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return remote;
}
__device__ __forceinline__ void tc_put(uint32_t at, uint32_t v) { asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
__device__ __forceinline__ void tc_put(uint32_t at, int v) { tc_put(at, (uint32_t)v); }
__device__ __forceinline__ void tc_put(uint32_t at, float v) { tc_put(at, __float_as_uint(v)); }
__device__ __forceinline__ void tc_put(uint32_t at, unsigned long long v) { asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(at), "l"(v) : "memory"); }
__device__ __forceinline__ void tc_put(uint32_t at, double v) { tc_put(at, (unsigned long long)__double_as_longlong(v)); }
__device__ __forceinline__ uint32_t tc_get(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
// By one warp: lane q to block q.
template <typename V>
__device__ __forceinline__ void tc_tell(V* mine, V v, int blocks) {
  if ((int)(threadIdx.x & 31) < blocks) tc_put(tc_there(mine, threadIdx.x & 31), v);
}
template <typename V>
__device__ __forceinline__ V tc_warp_sum(V v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <typename V>
__device__ __forceinline__ V tc_warp_scan(V v) {  // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V a = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += a;
  }
  return v;
}
__device__ __forceinline__ float tc_exp2(float x) {  // two steps of the last place
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kTcLog2e = 1.4426950408889634f;

// A row in shared memory and who looks at what: warp w has the columns [w * span, (w + 1) * span) of its block, four to a lane at a time.
struct TcRow {
  float* row;       // this block's adjusted logits; -inf behind its columns
  int v0, lo, hi;   // the block's first column; this warp's columns of the block, multiples of 128
  int rank, blocks;
  float m;
  float unit;       // log2(e) / temperature: z below is in units of ln 2
  float apart;      // the same, of a temperature of up to 64: places in the order keep apart what a higher one gives the same weight
  TcMail* mail;
  uint32_t* hist;   // counts, or upper and lower halves of weights
  float* list_l;    // a bin's tokens: logit, column
  int* list_at;
  // how far behind the largest logit
  __device__ __forceinline__ float behind(float l) const { return l == m ? 0.f : m - l; }
  __device__ __forceinline__ float z(float l) const { return __fmul_rn(behind(l), unit); }
  // a weight in steps of 2^-32 of the largest (which is one step short)
  __device__ __forceinline__ uint32_t steps(float z) const { return __float2uint_rn(tc_exp2(-z) * 4294967296.f); }
  __device__ __forceinline__ float place(float l) const { return __fmul_rn(behind(l), apart); }
  // no token with a smaller logit has a place (or with `per` unit, a z) up to this
  __device__ __forceinline__ float floor(float place, float per) const { return __fsub_rd(m, __fmul_ru(__fdiv_ru(place, per), 1.00001f)); }
  __device__ __forceinline__ float floor(float place) const { return floor(place, apart); }
  // f(column of the block, logit) of all, and of those that are not below a floor: few, where it cuts the bulk of a vocabulary off
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    for (int i = lo + 4 * (threadIdx.x & 31); i < hi; i += 128) {
      const float4 l = *reinterpret_cast<const float4*>(row + i);
      f(i, l.x);
      f(i + 1, l.y);
      f(i + 2, l.z);
      f(i + 3, l.w);
    }
  }
  template <typename F>
  __device__ __forceinline__ void each_above(float floor, F f) const {
    for (int i = lo + 4 * (threadIdx.x & 31); i < hi; i += 128) {
      const float4 l = *reinterpret_cast<const float4*>(row + i);
      if (fmaxf(fmaxf(l.x, l.y), fmaxf(l.z, l.w)) < floor) continue;
      if (!(l.x < floor)) f(i, l.x);
      if (!(l.y < floor)) f(i + 1, l.y);
      if (!(l.z < floor)) f(i + 2, l.z);
      if (!(l.w < floor)) f(i + 3, l.w);
    }
  }
};

// The last token that is kept: its logit and its column.
struct TcCut {
  bool on = false;
  float logit = 0.f;
  int at = 0;
  float floor = -INFINITY;  // no token below it is kept
  __device__ __forceinline__ bool keeps(const TcRow& c, int i, float l) const { return !on || l > logit || (l == logit && c.v0 + i <= at); }
};

// Tokens in order: the logit (not how far it is behind the largest, which rounding makes the same for some), then the column.
__device__ __forceinline__ unsigned long long tc_key(float l, int at) {
  const uint32_t u = __float_as_uint(__fadd_rn(l, 0.f));  // (one zero)
  return (unsigned long long)(u >> 31 ? u : ~u & 0x7fffffffu) << 32 | (uint32_t)at;
}
__device__ __forceinline__ uint32_t tc_key_of(float l) { return (uint32_t)(tc_key(l, 0) >> 32); }
__device__ __forceinline__ float tc_key_logit(unsigned long long key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float(u >> 31 ? u : ~u & 0x7fffffffu);
}
constexpr unsigned long long kTcNoKey = ~0ull;  // behind all
// Puts the num keys that lie in `keys` in ascending order, which has room for a power of two from 64 to twice the block's threads.  By all threads: a bitonic
// sort, a pair a thread; for pairs up to 32 apart a warp has its 64 keys to itself.  (Counting those in front of each instead took 140 us for 535
// tokens and 6 for 50.)
__device__ __forceinline__ void tc_sort(unsigned long long* keys, int num) {
  const int tid = threadIdx.x;
  int n = 64;
  while (n < num) n *= 2;
  for (int i = num + tid; i < n; i += kTcThreads) keys[i] = kTcNoKey;
  bool wide = true;  // the step before has been one of several warps
#pragma unroll 1
  for (int k = 2; k <= n; k <<= 1) {
#pragma unroll 1
    for (int j = k >> 1; j > 0; j >>= 1) {
      if (wide || j > 32) __syncthreads();
      else __syncwarp();
      wide = j > 32;
      if (tid >= n / 2) continue;
      const int i = 2 * tid - (tid & (j - 1));
      const unsigned long long a = keys[i], b = keys[i + j];
      if ((a > b) == ((i & k) == 0)) {
        keys[i] = b;
        keys[i + j] = a;
      }
    }
  }
  __syncthreads();
}

// What a step of a selection tells apart: bins of places, or, where those do not (tokens further behind than they reach, too many in the smallest bin), ten
// bits of the logits' keys at a time, so that in the end only equal logits are in one bin.
struct TcBins {
  bool keys = false;
  float base = 0.f, scale = kTcBins / 16.f;  // places
  int shift = 22, bits = 10;                 // keys: of those that begin with `prefix`
  uint32_t prefix = 0;
  // the token's bin, or one outside [0, kTcBins).  Differences of nearby places and products with powers of two are exact.
  __device__ __forceinline__ int of(const TcRow& c, float l) const {
    if (keys) {
      const uint32_t k = tc_key_of(l) >> shift;
      return k >> bits == prefix ? (int)(k & ((1u << bits) - 1)) : -1;
    }
    const float x = (c.place(l) - base) * scale;
    return x >= 0.f && x < (float)kTcBins ? (int)x : -1;
  }
};

// Where the cut lies that keeps the first `k` tokens (kMass false), or the shortest run with `p` of the weight (kMass true), of those that `had` keeps;
// off where nothing is cut.  By all threads of the cluster.  weighed: every block has told its tokens' weight.
template <bool kMass>
__device__ __forceinline__ TcCut tc_select(const TcRow& c, uint32_t k, float p, const TcCut& had, bool weighed) {
  constexpr int kWords = kMass ? 2 : 1;  // of a bin: its count, or its weight's halves
  TcMail& mail = *c.mail;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // places below 16; then up to 80; then down into a bin; then keys
  TcBins bins;
  float top = 16.f;
  int level = 0;
  unsigned long long before = 0;  // counts, or weights, in front of the bins
  double target = (double)k;
  const auto by_keys = [&]() {
    bins.keys = true;
    before = 0;
  };
#pragma unroll 1
  for (bool first = true;; first = false) {
    const bool weigh = kMass && first && !weighed;
    __syncthreads();  // (what was found before has been read)
    for (int i = tid; i < kWords * kTcBins; i += kTcThreads) c.hist[i] = 0;
    if (tid == 0) mail.listed = 0;
    __syncthreads();
    float weight = 0.f;
    c.each_above(weigh || bins.keys ? had.floor : fmaxf(had.floor, c.floor(top)), [&](int i, float l) {
      const float z = c.z(l);
      const int b = bins.of(c, l);
      if (!had.keeps(c, i, l)) return;
      if (weigh) weight += tc_exp2(-z);
      if (b < 0) return;
      if (kMass) {
        const uint32_t q = c.steps(z);
        atomicAdd(&c.hist[b], q >> 16);
        atomicAdd(&c.hist[kTcBins + b], q & 0xffffu);
      } else {
        atomicAdd(&c.hist[b], 1u);
      }
    });
    if (weigh) {
      weight = tc_warp_sum(weight);
      if (lane == 0) c.list_l[warp] = weight;  // (nothing is listed yet)
    }
    __syncthreads();
    if (weigh && warp == 0) tc_tell(&mail.weight[c.rank], tc_warp_sum(lane < kTcWarps ? c.list_l[lane] : 0.f), c.blocks);
    for (int i = warp; i < kTcCoarse; i += kTcWarps) {
      const int b = 32 * i + lane;  // (no sum of halves reaches 2^32: a block has fewer than 2^16 columns)
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        const uint32_t sum = __reduce_add_sync(0xffffffffu, c.hist[w * kTcBins + b]);
        if (lane == 0) mail.coarse[w][i] = sum;
      }
    }
    tc_cluster_sync();
    if (kMass && first) {
      float all = 0.f;
      for (int q = 0; q < c.blocks; ++q) all += mail.weight[q];
      target = fmax((double)p * (double)all * 4294967296., 0.5);
    }
    // the sum of bins, then the bin, that the cut lies in: every block for itself, a warp fetching from each
    const auto fetch = [&](const uint32_t* at, int apart) {  // at: this lane's place in a block
      if (warp < c.blocks) {
        uint32_t v[kWords];
#pragma unroll
        for (int w = 0; w < kWords; ++w) v[w] = tc_get(tc_there(at + w * apart, warp));
#pragma unroll
        for (int w = 0; w < kWords; ++w) mail.fetched[w][warp][lane] = v[w];
      }
      __syncthreads();
    };
    unsigned long long sum, upto;  // of counts or of weights
    const auto add_up = [&]() {
      sum = 0;
      for (int q = 0; q < c.blocks; ++q) {
        const unsigned long long upper = mail.fetched[0][q][lane];
        sum += kMass ? (upper << 16) + mail.fetched[kWords - 1][q][lane] : upper;
      }
      upto = before + tc_warp_scan(sum);
      return __ballot_sync(0xffffffffu, (double)upto >= target);
    };
    fetch(&mail.coarse[0][lane], kTcCoarse);
    unsigned hit = add_up();  // (by every warp alike)
    if (!hit) {
      before = __shfl_sync(0xffffffffu, upto, 31);
      tc_cluster_sync();  // (the blocks read this one's sums)
      // Fewer tokens, or less weight, than would be kept.  (A bin's parts have the bin's sums.)  Places that are weights: those below 2^-80 do not count.
      if (bins.keys || (bins.base > 0.f && c.apart == c.unit)) return TcCut();
      if (bins.base > 0.f) {
        by_keys();
      } else {
        bins.base = 16.f;
        bins.scale = kTcBins / 64.f;
        top = 80.f;
      }
      continue;
    }
    const int group = __ffs(hit) - 1;
    before = __shfl_sync(0xffffffffu, upto - sum, group);
    __syncthreads();  // (every warp has added up)
    fetch(c.hist + 32 * group + lane, kTcBins);
    hit = add_up();
    const int in_group = __ffs(hit) - 1, bin = 32 * group + in_group;
    const unsigned long long in_bin = __shfl_sync(0xffffffffu, sum, in_group);
    before = __shfl_sync(0xffffffffu, upto - sum, in_group);
    TcCut cut;
    cut.on = true;
    const float bin_floor = bins.keys ? had.floor : c.floor(bins.base + (float)(bin + 1) / bins.scale);
    const auto member = [&](int i, float l) { return bins.of(c, l) == bin && had.keeps(c, i, l); };
    // the bin's tokens: every block's own, then all of them where the histogram was
    c.each_above(bin_floor, [&](int i, float l) {
      if (!member(i, l)) return;
      const uint32_t at = atomicAdd(&mail.listed, 1u);
      if (at >= (uint32_t)kTcMembers) return;
      c.list_l[at] = l;
      c.list_at[at] = c.v0 + i;
    });
    __syncthreads();
    if (warp == 0) tc_tell(&mail.listed_by[c.rank], mail.listed, c.blocks);
    tc_cluster_sync();
    uint32_t members = 0;
    for (int q = 0; q < c.blocks; ++q) members += mail.listed_by[q];
    if (members <= (uint32_t)kTcMembers) {
      unsigned long long* keys = reinterpret_cast<unsigned long long*>(c.hist);
      const int num = (int)members;
      for (int i = tid; i < num; i += kTcThreads) {
        int q = 0;
        uint32_t at = i;
        while (at >= mail.listed_by[q]) at -= mail.listed_by[q++];
        const uint32_t l = tc_get(tc_there(c.list_l + at, q)), column = tc_get(tc_there(c.list_at + at, q));
        keys[i] = tc_key(__uint_as_float(l), (int)column);
      }
      tc_cluster_sync();  // (and nobody reads another block's list behind this)
      tc_sort(keys, num);
      if (kMass) {
        unsigned long long w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) w[i] = 2 * tid + i < num ? c.steps(c.z(tc_key_logit(keys[2 * tid + i]))) : 0;
        const unsigned long long upto_w = tc_warp_scan(w[0] + w[1]);
        unsigned long long* by_warp = reinterpret_cast<unsigned long long*>(c.list_l);
        if (lane == 31) by_warp[warp] = upto_w;
        __syncthreads();
        unsigned long long front = before + upto_w - w[0] - w[1];
        for (int v = 0; v < warp; ++v) front += by_warp[v];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (2 * tid + i < num && (double)front < target && (double)(front + w[i]) >= target) mail.cut = keys[2 * tid + i];
          front += w[i];
        }
        __syncthreads();
      }
      const unsigned long long key = kMass ? mail.cut : keys[k - (uint32_t)before - 1];
      cut.logit = cut.floor = tc_key_logit(key);
      cut.at = (int)(uint32_t)key;
      return cut;
    }
    if (!bins.keys || bins.shift > 0) {
      tc_cluster_sync();  // (the blocks read this one's bins)
      if (bins.keys) {  // bits 31 to 22, 21 to 12, 11 to 2, 1 and 0
        bins.prefix = bins.prefix << bins.bits | (uint32_t)bin;
        bins.bits = bins.shift < 10 ? bins.shift : 10;
        bins.shift -= bins.bits;
      } else if (level < 2) {
        top = bins.base + (float)(bin + 1) / bins.scale;
        bins.base += (float)bin / bins.scale;
        bins.scale *= (float)kTcBins;
        ++level;
      } else {
        by_keys();
      }
      continue;
    }
    // more equal logits than that: by index
    uint32_t want = k - (uint32_t)before;
    if (kMass) want = (uint32_t)fmin(fmax(ceil((target - (double)before) * members / fmax((double)in_bin, 1.)), 1.), (double)members);
    uint32_t mine = 0;
    c.each([&](int i, float l) { mine += member(i, l); });
    mine = tc_warp_sum(mine);
    uint32_t* tmp = reinterpret_cast<uint32_t*>(c.list_l);
    if (lane == 0) tmp[warp] = mine;
    __syncthreads();
    if (warp == 0) tc_tell(&mail.ties[c.rank], tc_warp_sum(lane < kTcWarps ? tmp[lane] : 0u), c.blocks);
    tc_cluster_sync();
    uint32_t passed = 0;
    for (int q = 0; q < c.rank; ++q) passed += mail.ties[q];
    for (int w = 0; w < warp; ++w) passed += tmp[w];
    if (passed < want && passed + mine >= want) {  // this warp has it
      for (int i0 = c.lo; i0 < c.hi; i0 += 128) {
        const int i = i0 + 4 * lane;
        const float4 l = *reinterpret_cast<const float4*>(c.row + i);
        const bool in[4] = {member(i, l.x), member(i + 1, l.y), member(i + 2, l.z), member(i + 3, l.w)};
        const uint32_t here = in[0] + in[1] + in[2] + in[3], there = tc_warp_scan(here), all = __shfl_sync(0xffffffffu, there, 31);
        if (passed < want && passed + all >= want) {
          uint32_t at = passed + there - here;
          for (int j = 0; j < 4; ++j)
            if (in[j] && ++at == want)
              for (int q = 0; q < c.blocks; ++q) tc_put(tc_there(&mail.cut_at, q), c.v0 + i + j);
        }
        passed += all;
      }
    }
    tc_cluster_sync();
    cut.logit = cut.floor = tc_key_logit((unsigned long long)(bins.prefix << bins.bits | (uint32_t)bin) << 32);
    cut.at = mail.cut_at;
    return cut;
  }
}

// vec: rows aligned to four elements
template <typename T>
__global__ void __launch_bounds__(kTcThreads, 2)
choose_tokens_kernel(const T* logits, long long stride, const TcRules r, const TcDraw d, int V, int cols, bool vec, bool append, long long* tokens,
                     float* logprobs, int32_t* status) {
  extern __shared__ __align__(16) uint8_t tc_smem[];
  __shared__ TcMail mail;
  __shared__ float tmp_f[kTcWarps];
  __shared__ int tmp_i[kTcWarps], tmp_n[kTcWarps];
  __shared__ double tmp_d[kTcWarps];
  __shared__ int tmp_s[kTcWarps];
  __shared__ unsigned long long tmp_u[kTcWarps];
  pdl_enter();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  TcRow c;
  c.rank = tc_rank();
  c.blocks = tc_size();
  const int e = blockIdx.x / c.blocks;
  const bool report = c.rank == 0;
  const TcEntry t = tc_entry(r, e, report && tid == 0, status);
  if (t.idle) {
    if (report && tid == 0) {
      tokens[e] = -1;
      logprobs[e] = -INFINITY;
    }
    return;
  }
  // no block writes to another one before that has begun
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n" ::: "memory");
  c.hist = reinterpret_cast<uint32_t*>(tc_smem);
  c.list_l = reinterpret_cast<float*>(c.hist + 3 * kTcBins);
  c.list_at = reinterpret_cast<int*>(c.list_l + kTcMembers);
  c.row = reinterpret_cast<float*>(tc_smem + kTcRowAt);
  c.mail = &mail;
  c.v0 = c.rank * cols;
  const int n = max(0, min(cols, V - c.v0)), padded = (n + 127) & ~127;
  const int span = ((padded >> 7) + kTcWarps - 1) / kTcWarps * 128;
  c.lo = min(padded, warp * span);
  c.hi = min(padded, c.lo + span);

  // ---- the row; its first columns on their way while the history is counted
  const T* src = logits + (long long)e * stride + c.v0;
  constexpr int kAhead = sizeof(T) == 2 ? 10 : 5;
  TcRaw<T> ahead[kAhead];
#pragma unroll
  for (int s = 0; s < kAhead; ++s) {
    const int i = 4 * (tid + s * kTcThreads);
    if (vec && i + 4 <= n) ahead[s].load(src + i);
  }
  uint32_t* table = reinterpret_cast<uint32_t*>(c.row);  // each place holds a count until its logit comes
  if (t.penalties) {
    for (int i = 4 * tid; i < padded; i += 4 * kTcThreads) *reinterpret_cast<uint4*>(table + i) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    tc_count(t, V, c.v0, n, table, report, status);
    __syncthreads();
  }
  float best = -INFINITY;
  const auto take = [&](int i, const TcRaw<T>& raw) {
    float f[4];
    if (vec && i + 4 <= n) {
      raw.get(f);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = i + j < n ? ld_fresh(src + i + j) : -INFINITY;
    }
    if (i < n) tc_settle(t, c.v0 + i, table + i, f);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[j] = fmaxf(f[j], -INFINITY);  // (not a number: no token)
      best = fmaxf(best, f[j]);
    }
    st_vec(c.row + i, f);
  };
#pragma unroll
  for (int s = 0; s < kAhead; ++s) {
    const int i = 4 * (tid + s * kTcThreads);
    if (i < padded) take(i, ahead[s]);
  }
  for (int i = 4 * (tid + kAhead * kTcThreads); i < padded; i += 4 * kTcThreads) {
    TcRaw<T> raw;
    if (vec && i + 4 <= n) raw.load(src + i);
    take(i, raw);
  }
  if (r.num_bias) {
    __syncthreads();
    tc_bias(r, t, e, V, c.v0, n, report, status, [&](int id, float s) { c.row[id - c.v0] = fmaxf(__fadd_rn(c.row[id - c.v0], s), -INFINITY); });
    __syncthreads();
    best = -INFINITY;
    for (int i = c.lo + 4 * lane; i < c.hi; i += 128) {
      const float4 l = *reinterpret_cast<const float4*>(c.row + i);
      best = fmaxf(best, fmaxf(fmaxf(l.x, l.y), fmaxf(l.z, l.w)));
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
  if (lane == 0) tmp_f[warp] = best;
  __syncthreads();
  asm volatile("barrier.cluster.wait.aligned;\n" ::: "memory");
  if (warp == 0) {
    best = lane < kTcWarps ? tmp_f[lane] : -INFINITY;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
    tc_tell(&mail.best[c.rank], best, c.blocks);
  }
  tc_cluster_sync();
  best = mail.best[0];
  for (int q = 1; q < c.blocks; ++q) best = fmaxf(best, mail.best[q]);
  c.m = best;
  if (best == -INFINITY) {  // nothing is allowed
    if (report && tid == 0) {
      tokens[e] = -1;
      logprobs[e] = -INFINITY;
    }
    return;
  }
  const float tau = d.temperature ? d.temperature[e] : 1.f;
  const int k = d.top_k ? d.top_k[e] : 0;
  const float p = d.top_p ? d.top_p[e] : 1.f, min_p = d.min_p ? d.min_p[e] : 0.f;
  const bool greedy = !(tau > 0.f) || k == 1;
  c.unit = greedy ? kTcLog2e : fminf(fmaxf(__fdiv_rn(kTcLog2e, tau), 1e-30f), 3e38f);  // (neither 0 nor infinite: products with infinity and 0 are numbers)
  c.apart = fmaxf(c.unit, kTcLog2e / 64.f);

  // ---- weights beside the largest ones', at temperature 1: a token's probability is exp(-behind) / (number of the largest + rest); and at the entry's
  float rest = 0.f, part = 0.f;
  int first = 0x7fffffff, equal = 0;
  const bool some = k > 0 && k < V, share = p < 1.f, cuts = some || share || min_p > 0.f;
  const bool in_reach = !greedy && cuts && (!some || k <= kTcShort * 3 / 4), by_places = in_reach && (some || share);
  const bool weighed = !greedy && !some && (share || !cuts), same_unit = c.unit == kTcLog2e;
  uint32_t* places = c.hist + 2 * kTcMembers;  // how many threads' largest logits are how far behind
  uint32_t* all_places = places + kTcPlaces;
  if (tid < kTcPlaces) places[tid] = 0;  // (nothing else has been there)
  float most = -INFINITY;
  for (int i0 = c.lo; i0 < c.hi; i0 += 128) {
    const int i = i0 + 4 * lane;
    const float4 l4 = *reinterpret_cast<const float4*>(c.row + i);
    const float l[4] = {l4.x, l4.y, l4.z, l4.w};
    const float top = fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3]));
    most = fmaxf(most, top);
    float far[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) far[j] = l[j] - c.m;
    if (top == c.m) {  // the largest are counted, and left out of the sums
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (l[j] == c.m) {
          first = min(first, c.v0 + i + j);
          ++equal;
          far[j] = -INFINITY;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) rest += tc_exp2(far[j] * kTcLog2e);
    if (weighed && !same_unit) {
#pragma unroll
      for (int j = 0; j < 4; ++j) part += tc_exp2(far[j] * c.unit);
    }
  }
  part = (same_unit ? rest : part) + (float)equal;
  double mine = tc_warp_sum((double)part);
  rest = tc_warp_sum(rest);
  equal = tc_warp_sum(equal);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
  if (lane == 0) {
    tmp_f[warp] = rest;
    tmp_i[warp] = first;
    tmp_n[warp] = equal;
    tmp_d[warp] = mine;
  }
  __syncthreads();
  if (by_places) {
    const float x = c.place(most) + 0.5f;
    if (x < 128.f) atomicAdd(&places[(__float_as_uint(x) >> 18) - (126u << 5)], 1u);
  }
  if (warp == 0) {
    rest = tc_warp_sum(lane < kTcWarps ? tmp_f[lane] : 0.f);
    equal = tc_warp_sum(lane < kTcWarps ? tmp_n[lane] : 0);
    first = lane < kTcWarps ? tmp_i[lane] : 0x7fffffff;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
    double block = 0.;
    for (int w = 0; w < kTcWarps; ++w) block += tmp_d[w];
    tc_tell(&mail.rest[c.rank], rest, c.blocks);
    tc_tell(&mail.equal[c.rank], equal, c.blocks);
    tc_tell(&mail.first[c.rank], first, c.blocks);
    tc_tell(&mail.mass[c.rank], block, c.blocks);
    tc_tell(&mail.weight[c.rank], (float)block, c.blocks);
  }

  // ---- few likely tokens: those from a floor on that at least as many are above as are looked for, since as many threads' largest are
  if (in_reach) {
    tc_cluster_sync();
    float reach = by_places ? 127.f : fmaxf(-log2f(min_p), 0.f) + 0.001f;
    if (by_places) {
      if (tid < kTcPlaces) {
        uint32_t sum = 0;
        for (int q = 0; q < c.blocks; ++q) sum += tc_get(tc_there(places + tid, q));
        all_places[tid] = sum;
      }
      __syncthreads();
      constexpr int kLane = kTcPlaces / 32;
      uint32_t of[kLane], sum = 0;
#pragma unroll
      for (int j = 0; j < kLane; ++j) sum += of[j] = all_places[kLane * lane + j];
      uint32_t upto = tc_warp_scan(sum) - sum;
      const uint32_t want = some ? (uint32_t)k : (uint32_t)kTcShare;
      int behind = kTcPlaces;
#pragma unroll
      for (int j = 0; j < kLane; ++j) {
        upto += of[j];
        if (behind == kTcPlaces && upto >= want) behind = kLane * lane + j + 1;
      }
      behind = __reduce_min_sync(0xffffffffu, behind);
      if (behind < kTcPlaces) reach = __uint_as_float(((126u << 5) + behind) << 18) - 0.5f;
    }
    const float floor = c.floor(reach, by_places ? c.apart : c.unit);
    int found = 0;  // by this warp, in order of the columns
    for (int i0 = c.lo; i0 < c.hi; i0 += 128) {
      const int i = i0 + 4 * lane;
      const float4 l4 = *reinterpret_cast<const float4*>(c.row + i);
      const float l[4] = {l4.x, l4.y, l4.z, l4.w};
      if (!__any_sync(0xffffffffu, fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3])) >= floor)) continue;
      const int here = (l[0] >= floor) + (l[1] >= floor) + (l[2] >= floor) + (l[3] >= floor), upto = tc_warp_scan(here);
      int at = found + upto - here;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (l[j] >= floor) {
          if (at < kTcShortWarp) {
            c.list_l[warp * kTcShortWarp + at] = l[j];
            c.list_at[warp * kTcShortWarp + at] = c.v0 + i + j;
          }
          ++at;
        }
      }
      found += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) tmp_s[warp] = found;
    __syncthreads();
    // this block's side by side
    float* own_l = reinterpret_cast<float*>(c.hist);
    int* own_at = reinterpret_cast<int*>(c.hist + kTcShort);
    const int by_warp = lane < kTcWarps ? tmp_s[lane] : 0, upto_warp = tc_warp_scan(by_warp), in_block = __shfl_sync(0xffffffffu, upto_warp, 31);
    const bool placed = !__any_sync(0xffffffffu, by_warp > kTcShortWarp) && in_block <= kTcShort;
    const bool by_share = share && !some;
    unsigned long long listed_mass = 0;
    if (placed) {
      const int at = __shfl_sync(0xffffffffu, upto_warp - by_warp, warp);
      for (int i = lane; i < found; i += 32) {
        const float l = c.list_l[warp * kTcShortWarp + i];
        own_l[at + i] = l;
        own_at[at + i] = c.list_at[warp * kTcShortWarp + i];
        if (by_share) listed_mass += c.steps(c.z(l));
      }
    }
    if (by_share) {
      listed_mass = tc_warp_sum(listed_mass);
      if (lane == 0) tmp_u[warp] = listed_mass;
      __syncthreads();
      if (warp == 0) tc_tell(&mail.listed_mass[c.rank], tc_warp_sum(lane < kTcWarps ? tmp_u[lane] : 0ull), c.blocks);
    }
    if (warp == 0) tc_tell(&mail.likely[c.rank], placed ? (uint32_t)in_block : kTcNoPlace, c.blocks);
    tc_cluster_sync();
    // every block finds out whether the cuts lie among them (the first k's weights are, if the first k are)
    uint32_t num = 0;
    for (int q = 0; q < c.blocks; ++q) num += mail.likely[q];
    bool ok = num > 0 && num <= (uint32_t)kTcShort && (!some || num >= (uint32_t)k || (reach >= 127.f && c.apart == c.unit));  // (weights below 2^-80 do not count)
    double target = INFINITY;
    if (by_share) {
      double of = 0.;
      listed_mass = 0;
      for (int q = 0; q < c.blocks; ++q) {
        of += mail.mass[q];
        listed_mass += mail.listed_mass[q];
      }
      target = fmax((double)(p > 0.f ? p : 0.f) * (of * 4294967296.), 0.5);
      ok = ok && (double)listed_mass >= target;
    }
    if (ok) {
      if (!report) {
        tc_cluster_sync();  // (the first block has this one's tokens)
        return;
      }
      // one a thread, in order of the columns
      float l = -INFINITY;
      int col = 0x7fffffff;
      if (tid < num) {
        int q = 0;
        uint32_t i = tid;
        while (i >= mail.likely[q]) i -= mail.likely[q++];
        const uint32_t raw = tc_get(tc_there(own_l + i, q));
        col = (int)tc_get(tc_there(own_at + i, q));
        l = __uint_as_float(raw);
      }
      __syncwarp();
      asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
      const float far = c.behind(l), w = tid < num ? tc_exp2(-__fmul_rn(far, c.unit)) : 0.f;
      const uint32_t q = tid < num ? __float2uint_rn(w * 4294967296.f) : 0u;
      // how many of them, and what weight, are in front of each (a weight beside the largest's alone needs no order)
      uint2* all = reinterpret_cast<uint2*>(c.list_l);
      all[tid] = make_uint2(__float_as_uint(l), q);
      __syncthreads();
      int place = 0;
      unsigned long long front_w = 0;
      if (by_places && tid < (int)num) {
#pragma unroll 4
        for (int j = 0; j < (int)num; ++j) {
          const uint2 other = all[j];
          const float other_l = __uint_as_float(other.x);
          if (other_l > l || (other_l == l && j < tid)) {
            ++place;
            front_w += other.y;
          }
        }
      }
      if (share && some) {
        if (tid < (int)num && place == min(k, (int)num) - 1) mail.some_mass = front_w + q;
        __syncthreads();
        target = fmax((double)(p > 0.f ? p : 0.f) * (double)mail.some_mass, 0.5);
      }
      const bool keep = tid < (int)num && (!some || place < k) && (double)front_w < target && w > 0.f && (w >= min_p || l == c.m);
      const double kept = keep ? (double)w : 0., upto_k = tc_warp_scan(kept);
      if (lane == 31) tmp_d[warp] = upto_k;
      __syncthreads();
      double from = 0., to = 0., sum = 0.;
      for (int w2 = 0; w2 < kTcWarps; ++w2) {
        if (w2 == warp) from = sum;
        sum += tmp_d[w2];
        if (w2 == warp) to = sum;
      }
      const float u = d.uniform ? d.uniform[e] : 0.f;
      const double goal = sum * (double)fminf(fmaxf(u, 0.f), 1.f - 5.9604645e-8f);
      // the first kept one that reaches beyond the goal (which is less than the sum)
      const unsigned hit = __ballot_sync(0xffffffffu, from + upto_k > goal);
      if (goal >= from && goal < to && lane == __ffs(hit) - 1) {
        double others = 0.;
        int same = 0;
        for (int b = 0; b < c.blocks; ++b) {
          others += mail.rest[b];
          same += mail.equal[b];
        }
        tokens[e] = col;
        logprobs[e] = -(float)((double)far + log1p(others + (same - 1)));
        if (append && t.history && t.length < r.capacity) r.history[(long long)t.slot * r.capacity + t.length] = col;
      }
      __syncwarp();
      asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
      return;
    }
  }

  TcCut by_count, by_mass;
  if (!greedy) {
    if (some) by_count = tc_select<false>(c, (uint32_t)k, 0.f, by_mass, false);
    if (share) by_mass = tc_select<true>(c, 0, p > 0.f ? p : 0.f, by_count, weighed);
  }
  int token = -1;
  float taken = 0.f;  // how far behind the largest it is
  if (greedy) {
    tc_cluster_sync();  // the other blocks' sums
    if (!report || tid != 0) return;
  } else {
    // ---- the kept weights, warp after warp in order of the columns
    const float floor = fmaxf(fmaxf(by_count.floor, by_mass.floor), min_p > 0.f ? c.floor(fmaxf(-log2f(min_p), 0.f) + 0.001f, c.unit) : -INFINITY);
    const auto weight = [&](int i, float l) {
      if (l < floor) return 0.f;
      const float w = tc_exp2(-c.z(l));
      return !cuts || ((w >= min_p || l == c.m) && by_mass.keeps(c, i, l) && by_count.keeps(c, i, l)) ? w : 0.f;
    };
    if (cuts) {
      part = 0.f;
      c.each_above(floor, [&](int i, float l) { part += weight(i, l); });
      mine = tc_warp_sum((double)part);
      __syncthreads();  // (the sums so far have been read)
      if (lane == 0) tmp_d[warp] = mine;
      __syncthreads();
      if (warp == 0) {
        double block = 0.;
        for (int w = 0; w < kTcWarps; ++w) block += tmp_d[w];
        tc_tell(&mail.mass[c.rank], block, c.blocks);
      }
    }
    tc_cluster_sync();
    double all = 0., from = 0., before = 0.;
    for (int q = 0; q < c.blocks; ++q) {
      if (q == c.rank) from = all;
      all += mail.mass[q];
    }
    // the warp that the goal falls to: each begins where the one in front ends
    for (int w = 0; w < warp; ++w) before += tmp_d[w];
    const double to = from + (before + mine);
    from += before;
    const float u = d.uniform ? d.uniform[e] : 0.f;
    const double goal = all * (double)fminf(fmaxf(u, 0.f), 1.f - 5.9604645e-8f);
    if (goal < from || goal >= to) return;
    for (int i0 = c.lo; i0 < c.hi; i0 += 128) {
      const int i = i0 + 4 * lane;
      const float4 l = *reinterpret_cast<const float4*>(c.row + i);
      const float f[4] = {l.x, l.y, l.z, l.w};
      float w[4], here = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = weight(i + j, f[j]);
        here += w[j];
      }
      const double upto = tc_warp_scan((double)here);
      double run = from + (upto - (double)here);
      int at = -1;
      float far = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        run += (double)w[j];
        if (w[j] > 0.f && at < 0 && run > goal) {
          at = c.v0 + i + j;
          far = c.behind(f[j]);
        }
      }
      const unsigned hit = __ballot_sync(0xffffffffu, at >= 0);
      if (hit) {
        token = __shfl_sync(0xffffffffu, at, __ffs(hit) - 1);
        taken = __shfl_sync(0xffffffffu, far, __ffs(hit) - 1);
        break;
      }
      from += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane != 0) return;
  }
  int largest = 0x7fffffff, same = 0;
  double others = 0.;
  for (int q = 0; q < c.blocks; ++q) {
    others += mail.rest[q];
    same += mail.equal[q];
    largest = min(largest, mail.first[q]);
  }
  if (token < 0) token = largest;  // (greedy, or the last bit of a sum)
  tokens[e] = token;
  logprobs[e] = -(float)((double)taken + log1p(others + (same - 1)));
  if (append && t.history && t.length < r.capacity) r.history[(long long)t.slot * r.capacity + t.length] = token;
}

}  // namespace b200kv

using namespace b200kv;

static int tc_rules(const b200dec_rules* r, int vocab, TcRules* d) {
  *d = TcRules{};
  if (!r) return B200KV_OK;
  if (r->num_bias < 0 || r->num_masks < 0 || r->capacity < 0 || r->num_histories < 0) return B200KV_E_RANGE;
  if (r->history && (!r->lengths || r->capacity < 1 || r->num_histories < 1)) return r->lengths ? B200KV_E_SHAPE : B200KV_E_NULL;
  if (r->num_bias && (!r->bias_ids || !r->bias)) return B200KV_E_NULL;
  if (r->masks && (!r->mask_rows || r->num_masks < 1)) return r->mask_rows ? B200KV_E_SHAPE : B200KV_E_NULL;
  if (r->masks && r->mask_words < (vocab + 31) / 32) return B200KV_E_SHAPE;
  const void* words[] = {r->history, r->slots, r->lengths, r->prompts, r->repetition, r->presence, r->frequency, r->bias_ids, r->bias, r->masks, r->mask_rows};
  for (const void* p : words)
    if (!aligned(p, 4)) return B200KV_E_ALIGN;
  *d = TcRules{r->history, r->slots, r->lengths, r->prompts, r->repetition, r->presence, r->frequency, r->bias_ids, r->bias, r->masks, r->mask_rows,
               r->capacity, r->num_histories, r->num_bias, r->num_masks, r->mask_words};
  return B200KV_OK;
}

extern "C" int b200dec_adjust_logits(const void* logits, int64_t stride, int32_t elem, const b200dec_rules* rules, float* out, int64_t out_stride,
                                     int32_t entries, int32_t vocab, int32_t* status, void* stream) {
  if (entries == 0) return B200KV_OK;
  if (!logits || !rules || !out) return B200KV_E_NULL;
  if (entries < 0 || entries > 65535 || vocab < 1) return B200KV_E_RANGE;
  if ((elem != 2 && elem != 4) || stride < vocab || out_stride < vocab) return B200KV_E_SHAPE;
  if (!aligned(logits, elem) || !aligned(out, 4)) return B200KV_E_ALIGN;
  if ((const void*)out == logits && (elem != 4 || stride != out_stride)) return B200KV_E_SHAPE;
  TcRules r;
  if (int rc = tc_rules(rules, vocab, &r)) return rc;
  const bool vec = aligned(logits, 4 * elem) && aligned(out, 16) && stride % 4 == 0 && out_stride % 4 == 0;
  // Fewer and longer blocks once there are nearly as many as multiprocessors all the same: each reads the whole history.  us, long and short blocks: 8 entries
  // of 151936 (80 long blocks) with histories of 1000 tokens 6.3 and 5.0, 64 of 32768 (128) with 8000 10.4 and 12.1 and with 1000 the same, 32 of 151936
  // (320) 10.5 and 11.4.
  const bool wide = (long long)entries * ((vocab + 8 * kAjCols - 1) / (8 * kAjCols)) * 4 >= (long long)device_sms() * 3;
  const int cols = wide ? 8 * kAjCols : 2 * kAjCols;
  const dim3 grid((unsigned)((vocab + cols - 1) / cols), (unsigned)entries);
  auto go = [&](auto kernel, auto* src) {
    if (!allow_smem(kernel, 8 * kAjCols * 4)) return launch_result(cudaErrorInvalidValue);
    return launch_result(launch_kernel(take_early_launch((cudaStream_t)stream), kernel, grid, dim3(kAjThreads), (size_t)cols * 4, (cudaStream_t)stream, src,
                                       (long long)stride, r, out, (long long)out_stride, (int)vocab, vec, status));
  };
  if (elem == 4) return wide ? go(adjust_logits_kernel<float, 8>, (const float*)logits) : go(adjust_logits_kernel<float, 2>, (const float*)logits);
  return wide ? go(adjust_logits_kernel<uint16_t, 8>, (const uint16_t*)logits) : go(adjust_logits_kernel<uint16_t, 2>, (const uint16_t*)logits);
}

extern "C" int b200dec_choose_tokens(const void* logits, int64_t stride, int32_t elem, const b200dec_rules* rules, const b200dec_draw* draw,
                                     int32_t entries, int32_t vocab, int32_t append, int64_t* tokens, float* logprobs, int32_t* status,
                                     void* stream) {
  if (entries == 0) return B200KV_OK;
  if (!logits || !draw || !tokens || !logprobs) return B200KV_E_NULL;
  if (draw->temperature && !draw->uniform) return B200KV_E_NULL;
  if (entries < 0 || entries > (1 << 24) || vocab < 1 || vocab > kTcMaxCluster * kTcMaxLocal) return B200KV_E_RANGE;
  if ((elem != 2 && elem != 4) || stride < vocab) return B200KV_E_SHAPE;
  if (!aligned(logits, elem) || !aligned(tokens, 8) || !aligned(logprobs, 4)) return B200KV_E_ALIGN;
  const void* numbers[] = {draw->temperature, draw->top_k, draw->top_p, draw->min_p, draw->uniform};
  for (const void* p : numbers)
    if (!aligned(p, 4)) return B200KV_E_ALIGN;
  TcRules r;
  if (int rc = tc_rules(rules, vocab, &r)) return rc;
  const TcDraw d{draw->temperature, draw->top_k, draw->top_p, draw->min_p, draw->uniform};
  // Halved while that leaves a block few columns, or more blocks than are resident at once (two a multiprocessor, but for what clusters of eight leave of a
  // graphics cluster), and two blocks still share a multiprocessor.  us with 8, 4, 2 and 1 blocks, 50 and 0.9 kept of 32768: one entry 12.8, 13.3, 15.8 and
  // 20.1, 32 entries 15.5, 14.0, 15.8 and 20.0, 64 entries 29, 16.2, 16.0 and 20.1, 128 entries 56, 31, 19 and 20; of 8000, 256 entries 103, 51, 29 and 17;
  // 64 entries of 151936 with 8 and 4 (one block a multiprocessor) 37 and 41.
  int blocks = kTcMaxCluster;
  const auto share = [&](int n) { return ((vocab + n - 1) / n + 127) / 128 * 128; };
  const auto resident = [&](int n) { return (long long)entries * n <= device_sms() * (n == 8 ? 12 : 12.25) / 7; };
  while (blocks > 1 && share(blocks / 2) <= 20 * 1024 && (share(blocks) < 2048 || !resident(blocks))) blocks /= 2;
  const int cols = share(blocks);
  const bool vec = aligned(logits, 4 * elem) && stride % 4 == 0;
  auto go = [&](auto kernel, auto* src) {
    if (!allow_smem(kernel, kTcRowAt + kTcMaxLocal * 4)) return launch_result(cudaErrorInvalidValue);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(entries * blocks));
    cfg.blockDim = dim3(kTcThreads);
    cfg.dynamicSmemBytes = kTcRowAt + (size_t)cols * 4;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = blocks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = take_early_launch((cudaStream_t)stream) ? 2 : 1;
    return launch_result(cudaLaunchKernelEx(&cfg, kernel, src, (long long)stride, r, d, (int)vocab, cols, vec, append != 0, (long long*)tokens,
                                            logprobs, status));
  };
  return elem == 4 ? go(choose_tokens_kernel<float>, (const float*)logits) : go(choose_tokens_kernel<uint16_t>, (const uint16_t*)logits);
}
