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
// A cut is found by histograms of z (counts, and weights as integers, so that no order of additions matters), down to the few tokens of
// one bin, which are put in order by comparison.
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
  bool bad = false;
  t.slot = r.slots ? r.slots[e] : e;
  t.idle = t.slot < 0;
  if (t.slot < -1 || (r.history && t.slot >= r.num_histories)) { bad = true; t.idle = true; }
  t.length = t.prompt = 0;
  t.history = nullptr;
  if (r.history && !t.idle) {
    t.length = r.lengths[e];
    t.prompt = r.prompts ? r.prompts[e] : t.length;
    if (t.length < 0 || t.length > r.capacity || t.prompt < 0) bad = true;
    t.length = max(0, min(t.length, r.capacity));
    t.prompt = max(0, t.prompt);
    t.history = r.history + (long long)t.slot * r.capacity;
  }
  t.repetition = r.repetition ? r.repetition[e] : 1.f;
  t.presence = r.presence ? r.presence[e] : 0.f;
  t.frequency = r.frequency ? r.frequency[e] : 0.f;
  t.penalties = t.length > 0 && (t.repetition != 1.f || t.presence != 0.f || t.frequency != 0.f);
  t.mask = nullptr;
  if (r.masks && r.mask_rows) {
    const int m = r.mask_rows[e];
    if (m >= 0 && m < r.num_masks) t.mask = r.masks + (long long)m * r.mask_words;
    else if (m != -1) bad = true;
  }
  if (bad && report && status) atomicOr(status, B200KV_S_BAD_POSITION);
  return t;
}

constexpr uint32_t kTcSeen = 0x80000000u;  // beside how often a token stands in the output

// table[v - v0] for the columns v0 .. v0 + n of this block; cleared by the caller, with a barrier on both sides.
__device__ __forceinline__ void tc_count(const TcEntry& t, int V, int v0, int n, uint32_t* table, bool report, int32_t* status) {
  auto take = [&](int i, int id) {
    const int at = id - v0;
    if (at >= 0 && at < n) {
      if (i >= t.prompt) atomicAdd(&table[at], 1u);
      atomicOr(&table[at], kTcSeen);
    }
    if (report && (id < 0 || id >= V) && status) atomicOr(status, B200KV_S_BAD_POSITION);
  };
  const int head = min(t.length, (int)((16 - (reinterpret_cast<uintptr_t>(t.history) & 15)) & 15) / 4);
  if ((int)threadIdx.x < head) take(threadIdx.x, t.history[threadIdx.x]);
  const int quads = (t.length - head) / 4;
  for (int i = threadIdx.x; i < quads; i += blockDim.x) {
    const int4 q = __ldcg(reinterpret_cast<const int4*>(t.history + head) + i);
    take(head + 4 * i, q.x);
    take(head + 4 * i + 1, q.y);
    take(head + 4 * i + 2, q.z);
    take(head + 4 * i + 3, q.w);
  }
  const int rest = head + 4 * quads + threadIdx.x;
  if (rest < t.length) take(rest, t.history[rest]);
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

// kN logits from column v on (aligned to their size)
template <typename T, int kN>
__device__ __forceinline__ void tc_load(const T* p, float (&f)[kN]) { ld_vec(p, f); }

// ---------------------------------------------------------------------------------------------------------------- adjusted logits
constexpr int kAjThreads = 256;
constexpr int kAjCols = 4096;  // of a block

// grid (ceil(V / kAjCols), entries).  kVec: 8 columns of a thread at a time, rows aligned to 16 bytes on both sides.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kAjThreads)
adjust_logits_kernel(const T* logits, long long stride, const TcRules r, float* out, long long out_stride, int V, int32_t* status) {
  __shared__ uint32_t table[kAjCols];
  pdl_enter();
  pdl_wait();
  const int e = blockIdx.y, v0 = blockIdx.x * kAjCols, n = min(kAjCols, V - v0), tid = threadIdx.x;
  const bool report = blockIdx.x == 0;
  const TcEntry t = tc_entry(r, e, report && tid == 0, status);
  if (t.idle) return;
  if (t.penalties) {
    for (int i = tid; i < kAjCols; i += kAjThreads) table[i] = 0;
    __syncthreads();
    tc_count(t, V, v0, n, table, report, status);
    __syncthreads();
  }
  const T* src = logits + (long long)e * stride + v0;
  float* dst = out + (long long)e * out_stride + v0;
  constexpr int kN = kVec ? 8 : 1;
  for (int i = tid * kN; i < n; i += kAjThreads * kN) {
    if (kVec && i + kN > n) {
      for (int j = i; j < n; ++j) {
        const float l = tc_penalised(t, ld_elem(src + j), t.penalties ? table[j] : 0u);
        dst[j] = tc_allowed(t, v0 + j) ? l : -INFINITY;
      }
      break;
    }
    float f[kN];
    tc_load<T, kN>(src + i, f);
    const uint32_t bits = t.mask ? t.mask[(v0 + i) >> 5] >> ((v0 + i) & 31) : ~0u;
#pragma unroll
    for (int j = 0; j < kN; ++j) {
      if (t.penalties) f[j] = tc_penalised(t, f[j], table[i + j]);
      if (!(bits >> j & 1u)) f[j] = -INFINITY;
    }
    st_vec(dst + i, f);
  }
  if (r.num_bias) {
    __syncthreads();  // what the block's other threads wrote
    tc_bias(r, t, e, V, v0, n, report, status, [&](int id, float s) { dst[id - v0] = __fadd_rn(dst[id - v0], s); });
  }
}

// ---------------------------------------------------------------------------------------------------------------- the choice
constexpr int kTcThreads = 512;
constexpr int kTcWarps = kTcThreads / 32;
constexpr int kTcCluster = 8;
constexpr int kTcBins = 2048;
constexpr int kTcPerRank = kTcBins / kTcCluster;
constexpr float kTcBinsPerUnit = 64.f;  // of z: 32 units in all, behind which a token's weight is below 1.3e-14
constexpr int kTcMembers = 2048;        // tokens of one bin that are put in order
constexpr int kTcMaxLocal = 48 * 1024;  // columns of a block
constexpr uint32_t kTcHistBytes = kTcBins * 12;
static_assert(kTcMembers * 12 <= kTcHistBytes, "a bin's tokens take the place of the histogram");

struct TcDraw {
  const float* temperature;
  const int32_t* top_k;
  const float *top_p, *min_p, *uniform;
};

// What the blocks of a cluster tell one another; every block has a copy of its own.
struct TcMail {
  float best[kTcCluster];
  int best_at[kTcCluster];
  double rest[kTcCluster], mass[kTcCluster];
  unsigned long long bin_mass[kTcCluster];
  uint32_t bin_count[kTcCluster];
  uint32_t found;  // 1: this bin, 2: the cut lies behind all tokens, 3: among tokens of no weight
  int bin;
  uint32_t count_before, members;
  unsigned long long mass_before, mass_all;
  float cut_behind;
  int cut_at;
  uint32_t listed;
  uint32_t ties[kTcCluster];
};

__device__ __forceinline__ uint32_t tc_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void tc_cluster_sync() {
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
template <typename V>
__device__ __forceinline__ void tc_tell(V* mine, V v) {  // by one thread, to every block
#pragma unroll
  for (int q = 0; q < kTcCluster; ++q) tc_put(tc_there(mine, q), v);
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
// Sums over the threads in front of this one (what the thread in front of it has for `upto`) and up to it; `all`: over the block.  tmp: one value
// per warp.
template <typename V>
__device__ __forceinline__ V tc_block_before(V v, V* tmp, V& upto, V& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const V s = tc_warp_scan(v);
  const V prev = __shfl_up_sync(0xffffffffu, s, 1);
  if (lane == 31) tmp[warp] = s;
  __syncthreads();
  V before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kTcWarps; ++w) {
    if (w == warp) before = total;
    total += tmp[w];
  }
  __syncthreads();
  all = total;
  upto = before + s;
  return before + (lane ? prev : (V)0);
}

struct TcRow {
  float* row;   // this block's adjusted logits
  int v0, n;    // its columns
  int lo, hi;   // this thread's, of the block
  int rank;
  float m, inv_tau;
  TcMail* mail;
  uint32_t* hist;  // counts, upper and lower halves of weights
  double* tmp;     // kTcWarps
  // how far behind the largest logit, in units of the temperature
  __device__ __forceinline__ float behind(float l) const { return l == m ? 0.f : m - l; }
  __device__ __forceinline__ float z(float l) const { return __fmul_rn(behind(l), inv_tau); }
  // a weight in steps of 2^-32 of the largest (which is one step short)
  __device__ __forceinline__ uint32_t steps(float z) const { return __float2uint_rn(expf(-z) * 4294967296.f); }
};

// A bin of z, and the last token that is kept: of all (exact: how far it is behind the largest, and its column), or of the bin's (its column).
struct TcCut {
  bool exact;
  float behind;
  int at;
  float base, scale;
  int bin, level;
  // -1: in front of the bin, 0: in it, 1: behind it.  Differences of nearby values and products with powers of two are exact.
  __device__ __forceinline__ int side(float z) const {
    const float x = (z - base) * scale;
    if (level && !(x >= 0.f && x < (float)kTcBins)) return x < 0.f ? -1 : 1;
    const int b = x < (float)(kTcBins - 1) ? (int)x : kTcBins - 1;
    return b < bin ? -1 : b > bin;
  }
};

// Where the cut lies that keeps the first `k` tokens (kMass false), or the shortest run with `p` of the weight (kMass true); false: nothing is cut.
// By all threads of the cluster.
template <bool kMass>
__device__ bool tc_select(const TcRow& c, uint32_t k, float p, TcCut& cut) {
  TcMail& mail = *c.mail;
  const int tid = threadIdx.x;
  float base = 0.f, scale = kTcBinsPerUnit;
  uint32_t count_before = 0;
  unsigned long long mass_before = 0;
  double target = 0.;
  for (int level = 0;; ++level) {
    __syncthreads();  // (what was told before has been read)
    for (int i = tid; i < 3 * kTcBins; i += kTcThreads) c.hist[i] = 0;
    if (tid == 0) {
      mail.found = 0;
      mail.listed = 0;
    }
    __syncthreads();
    for (int i = c.lo; i < c.hi; ++i) {
      const float l = c.row[i];
      if (l == -INFINITY) continue;
      const float z = c.z(l), at = (z - base) * scale;
      if (level && !(at >= 0.f && at < (float)kTcBins)) continue;
      const int b = at < (float)(kTcBins - 1) ? (int)at : kTcBins - 1;
      atomicAdd(&c.hist[b], 1u);
      if (kMass) {
        const uint32_t q = c.steps(z);
        atomicAdd(&c.hist[kTcBins + b], q >> 16);
        atomicAdd(&c.hist[2 * kTcBins + b], q & 0xffffu);
      }
    }
    tc_cluster_sync();
    // this block's share of the bins, over all blocks
    uint32_t count = 0;
    unsigned long long mass = 0;
    if (tid < kTcPerRank) {
      const uint32_t* mine = c.hist + c.rank * kTcPerRank + tid;
#pragma unroll
      for (int q = 0; q < kTcCluster; ++q) {
        count += tc_get(tc_there(mine, q));
        if (kMass) mass += ((unsigned long long)tc_get(tc_there(mine + kTcBins, q)) << 16) + tc_get(tc_there(mine + 2 * kTcBins, q));
      }
    }
    uint32_t block_count, unused_count;
    unsigned long long block_mass = 0, m_before = 0, unused_mass;
    uint32_t c_before = tc_block_before(count, reinterpret_cast<uint32_t*>(c.tmp), unused_count, block_count);
    if (kMass) m_before = tc_block_before(mass, reinterpret_cast<unsigned long long*>(c.tmp), unused_mass, block_mass);
    if (tid == 0) {
      tc_tell(&mail.bin_count[c.rank], block_count);
      if (kMass) tc_tell(&mail.bin_mass[c.rank], block_mass);
    }
    tc_cluster_sync();
    uint32_t all_count = 0;
    unsigned long long all_mass = 0;
    c_before += count_before;
    m_before += mass_before;
    for (int q = 0; q < kTcCluster; ++q) {
      if (q < c.rank) {
        c_before += mail.bin_count[q];
        if (kMass) m_before += mail.bin_mass[q];
      }
      all_count += mail.bin_count[q];
      if (kMass) all_mass += mail.bin_mass[q];
    }
    if (level == 0) {
      if (!kMass && all_count <= k) return false;
      if (kMass) target = fmax((double)p * (double)all_mass, 0.5);
    }
    // the bin that the cut lies in
    const bool here = kMass ? (double)m_before < target && (double)(m_before + mass) >= target : c_before < k && c_before + count >= k;
    if (tid < kTcPerRank && here && count) {
      const int b = c.rank * kTcPerRank + tid;
      tc_tell(&mail.bin, b);
      tc_tell(&mail.count_before, c_before);
      tc_tell(&mail.mass_before, m_before);
      tc_tell(&mail.mass_all, mass);
      tc_tell(&mail.members, count);
      tc_tell(&mail.found, level == 0 && b == kTcBins - 1 ? 3u : 1u);
    }
    tc_cluster_sync();
    if (!mail.found) return false;
    cut = TcCut{false, 0.f, -1, base, scale, mail.bin, level};
    if (mail.found == 3) return true;  // every token in front of the last bin is kept, those in it have no weight
    const uint32_t members = mail.members;
    count_before = mail.count_before;
    mass_before = mail.mass_before;
    auto member = [&](float l) { return l != -INFINITY && cut.side(c.z(l)) == 0; };
    if (members <= kTcMembers) {
      // to block 0, whose histogram is read by nobody any more: how far behind, column and weight
      for (int i = c.lo; i < c.hi; ++i) {
        const float l = c.row[i];
        if (!member(l)) continue;
        uint32_t at;
        asm volatile("atom.shared::cluster.add.u32 %0, [%1], 1;" : "=r"(at) : "r"(tc_there(&mail.listed, 0)) : "memory");
        if (at >= (uint32_t)kTcMembers) continue;
        tc_put(tc_there(c.hist + at, 0), c.behind(l));
        tc_put(tc_there(c.hist + kTcMembers + at, 0), c.v0 + i);
        if (kMass) tc_put(tc_there(c.hist + 2 * kTcMembers + at, 0), c.steps(c.z(l)));
      }
      tc_cluster_sync();
      if (c.rank == 0) {
        const uint32_t num = min(mail.listed, (uint32_t)kTcMembers);
        const float* far = reinterpret_cast<const float*>(c.hist);
        const int* at = reinterpret_cast<const int*>(c.hist + kTcMembers);
        const uint32_t* w = c.hist + 2 * kTcMembers;
        for (uint32_t i = tid; i < num; i += kTcThreads) {
          uint32_t before = 0;
          unsigned long long weight = 0;
          for (uint32_t j = 0; j < num; ++j) {
            if (far[j] < far[i] || (far[j] == far[i] && at[j] < at[i])) {
              ++before;
              if (kMass) weight += w[j];
            }
          }
          const bool last = kMass ? (double)(mass_before + weight) < target && (double)(mass_before + weight + w[i]) >= target : count_before + before + 1 == k;
          if (last) {
            tc_tell(&mail.cut_behind, far[i]);
            tc_tell(&mail.cut_at, at[i]);
          }
        }
      }
      tc_cluster_sync();
      cut.exact = true;
      cut.behind = mail.cut_behind;
      cut.at = mail.cut_at;
      return true;
    }
    if (level < 2) {
      base += (float)mail.bin / scale;
      scale *= (float)kTcBins;
      continue;
    }
    // more tokens than that within 2^-28 of one another: equal ones, by index
    uint32_t want = kMass ? (uint32_t)fmin(fmax(ceil((target - (double)mass_before) * members / fmax((double)mail.mass_all, 1.)), 1.), (double)members) : k - count_before;
    uint32_t mine = 0, upto, block;
    for (int i = c.lo; i < c.hi; ++i) mine += member(c.row[i]);
    uint32_t before = tc_block_before(mine, reinterpret_cast<uint32_t*>(c.tmp), upto, block);
    if (tid == 0) tc_tell(&mail.ties[c.rank], block);
    tc_cluster_sync();
    for (int q = 0; q < c.rank; ++q) before += mail.ties[q];
    if (before < want && before + mine >= want) {
      for (int i = c.lo; i < c.hi; ++i) {
        if (member(c.row[i]) && ++before == want) tc_tell(&mail.cut_at, c.v0 + i);
      }
    }
    tc_cluster_sync();
    cut.at = mail.cut_at;
    return true;
  }
}

template <typename T, bool kVec>
__global__ void __launch_bounds__(kTcThreads)
choose_tokens_kernel(const T* logits, long long stride, const TcRules r, const TcDraw d, int V, int cols, int seg, bool append, long long* tokens,
                     float* logprobs, int32_t* status) {
  extern __shared__ __align__(16) uint8_t tc_smem[];
  __shared__ TcMail mail;
  __shared__ double tmp[kTcWarps];
  __shared__ float tmp_v[kTcWarps];
  __shared__ int tmp_i[kTcWarps];
  pdl_enter();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  TcRow c;
  c.rank = (int)tc_rank();
  const int e = blockIdx.x / kTcCluster;
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
  c.row = reinterpret_cast<float*>(tc_smem + kTcHistBytes);
  c.mail = &mail;
  c.tmp = tmp;
  c.v0 = c.rank * cols;
  c.n = max(0, min(cols, V - c.v0));
  c.lo = min(c.n, tid * seg);
  c.hi = min(c.n, c.lo + seg);

  // ---- the row
  uint32_t* table = reinterpret_cast<uint32_t*>(c.row);  // each place holds a count until its logit comes
  if (t.penalties) {
    for (int i = tid; i < c.n; i += kTcThreads) table[i] = 0;
    __syncthreads();
    tc_count(t, V, c.v0, c.n, table, report, status);
    __syncthreads();
  }
  const T* src = logits + (long long)e * stride + c.v0;
  constexpr int kN = kVec ? 8 : 1;
  for (int i = tid * kN; i < c.n; i += kTcThreads * kN) {
    float f[kN];
    const bool whole = i + kN <= c.n;
    if (whole) {
      tc_load<T, kN>(src + i, f);
    } else {
#pragma unroll
      for (int j = 0; j < kN; ++j) f[j] = i + j < c.n ? ld_elem(src + i + j) : 0.f;
    }
    const uint32_t bits = t.mask ? t.mask[(c.v0 + i) >> 5] >> ((c.v0 + i) & 31) : ~0u;
    float seen[kN];
    if (t.penalties) {
      if (whole) tc_load<float, kN>(c.row + i, seen);
      else
#pragma unroll
        for (int j = 0; j < kN; ++j) seen[j] = i + j < c.n ? c.row[i + j] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < kN; ++j) {
      if (t.penalties) f[j] = tc_penalised(t, f[j], __float_as_uint(seen[j]));
      if (!(bits >> j & 1u) || f[j] != f[j]) f[j] = -INFINITY;
    }
    if (whole) st_vec(c.row + i, f);
    else
#pragma unroll
      for (int j = 0; j < kN; ++j)
        if (i + j < c.n) c.row[i + j] = f[j];
  }
  __syncthreads();
  if (r.num_bias) {
    tc_bias(r, t, e, V, c.v0, c.n, report, status, [&](int id, float s) {
      const float l = __fadd_rn(c.row[id - c.v0], s);
      c.row[id - c.v0] = l == l ? l : -INFINITY;
    });
    __syncthreads();
  }

  // ---- the largest, the first one of equals
  float best = -INFINITY;
  int at = 0x7fffffff;
  for (int i = c.lo; i < c.hi; ++i)
    if (c.row[i] > best) { best = c.row[i]; at = c.v0 + i; }
  auto better = [&](float v, int i) {
    if (v > best || (v == best && i < at)) { best = v; at = i; }
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) better(__shfl_xor_sync(0xffffffffu, best, o), __shfl_xor_sync(0xffffffffu, at, o));
  if (lane == 0) { tmp_v[warp] = best; tmp_i[warp] = at; }
  __syncthreads();
  asm volatile("barrier.cluster.wait.aligned;\n" ::: "memory");
  if (tid == 0) {
    for (int w = 1; w < kTcWarps; ++w) better(tmp_v[w], tmp_i[w]);
    tc_tell(&mail.best[c.rank], best);
    tc_tell(&mail.best_at[c.rank], at);
  }
  tc_cluster_sync();
  best = mail.best[0];
  at = mail.best_at[0];
  for (int q = 1; q < kTcCluster; ++q) better(mail.best[q], mail.best_at[q]);
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
  c.inv_tau = greedy ? 1.f : fminf(__fdiv_rn(1.f, tau), 3e38f);  // (finite: the largest is 0 units behind itself)

  // ---- weights beside the largest's, at temperature 1: the token's probability is exp(-behind) / (1 + rest)
  float rest = 0.f;
  for (int i = c.lo; i < c.hi; ++i)
    if (c.v0 + i != at) rest += expf(-c.behind(c.row[i]));
  double block_rest, unused;
  tc_block_before((double)rest, tmp, unused, block_rest);
  if (tid == 0) tc_tell(&mail.rest[c.rank], block_rest);

  if (!greedy) {
    TcCut cut;
    auto apply = [&]() {
      for (int i = c.lo; i < c.hi; ++i) {
        const float l = c.row[i], far = c.behind(l);
        const int side = cut.exact ? (far < cut.behind ? -1 : far > cut.behind) : cut.side(c.z(l));
        if (side > 0 || (side == 0 && c.v0 + i > cut.at)) c.row[i] = -INFINITY;
      }
    };
    if (k > 0 && k < V && tc_select<false>(c, (uint32_t)k, 0.f, cut)) apply();
    if (p < 1.f && tc_select<true>(c, 0, p > 0.f ? p : 0.f, cut)) apply();
  }
  int token = at;
  float taken = 0.f;  // how far behind the largest it is
  if (greedy) {
    tc_cluster_sync();  // the other blocks' rests
    if (!report || tid != 0) return;
  } else {
    // ---- the kept weights, thread after thread in order of the columns
    auto weight = [&](int i) {
      const float l = c.row[i];
      if (l == -INFINITY) return 0.f;
      const float w = expf(-c.z(l));
      return w >= min_p || l == c.m ? w : 0.f;
    };
    float mine = 0.f;
    for (int i = c.lo; i < c.hi; ++i) mine += weight(i);
    double block, upto;
    const double before = tc_block_before((double)mine, tmp, upto, block);
    if (tid == 0) tc_tell(&mail.mass[c.rank], block);
    tc_cluster_sync();
    double all = 0., start = 0.;
    for (int q = 0; q < kTcCluster; ++q) {
      if (q == c.rank) start = all;
      all += mail.mass[q];
    }
    // the thread that the goal falls to (each begins where the one in front ends); its own sums, as above, say which column
    const float u = d.uniform ? d.uniform[e] : 0.f;
    const double goal = all * (double)fminf(fmaxf(u, 0.f), 1.f - 5.9604645e-8f), from = start + before;
    if (goal < from || goal >= start + upto) return;
    float sum = 0.f;
    for (int i = c.lo; i < c.hi; ++i) {
      const float w = weight(i);
      sum += w;
      if (w > 0.f) {
        token = c.v0 + i;
        taken = c.behind(c.row[i]);
      }
      if (from + (double)sum > goal) break;
    }
  }
  double others = 0.;
  for (int q = 0; q < kTcCluster; ++q) others += mail.rest[q];
  tokens[e] = token;
  logprobs[e] = -(float)((double)taken + log1p(others));
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
  const dim3 grid((unsigned)((vocab + kAjCols - 1) / kAjCols), (unsigned)entries);
  const bool vec = aligned(logits, 16) && aligned(out, 16) && stride * elem % 16 == 0 && out_stride % 4 == 0;
  cudaStream_t s = (cudaStream_t)stream;
  auto go = [&](auto kernel, auto* src) { return launch_result(launch_chained(kernel, grid, dim3(kAjThreads), 0, s, src, (long long)stride, r, out, (long long)out_stride, (int)vocab, status)); };
  if (elem == 4) return vec ? go(adjust_logits_kernel<float, true>, (const float*)logits) : go(adjust_logits_kernel<float, false>, (const float*)logits);
  return vec ? go(adjust_logits_kernel<uint16_t, true>, (const uint16_t*)logits) : go(adjust_logits_kernel<uint16_t, false>, (const uint16_t*)logits);
}

extern "C" int b200dec_choose_tokens(const void* logits, int64_t stride, int32_t elem, const b200dec_rules* rules, const b200dec_draw* draw,
                                     int32_t entries, int32_t vocab, int32_t append, int64_t* tokens, float* logprobs, int32_t* status,
                                     void* stream) {
  if (entries == 0) return B200KV_OK;
  if (!logits || !draw || !tokens || !logprobs) return B200KV_E_NULL;
  if (draw->temperature && !draw->uniform) return B200KV_E_NULL;
  if (entries < 0 || entries > (1 << 24) || vocab < 1 || vocab > kTcCluster * kTcMaxLocal) return B200KV_E_RANGE;
  if ((elem != 2 && elem != 4) || stride < vocab) return B200KV_E_SHAPE;
  if (!aligned(logits, elem) || !aligned(tokens, 8) || !aligned(logprobs, 4)) return B200KV_E_ALIGN;
  for (const void* p : {(const void*)draw->temperature, (const void*)draw->top_k, (const void*)draw->top_p, (const void*)draw->min_p, (const void*)draw->uniform})
    if (!aligned(p, 4)) return B200KV_E_ALIGN;
  TcRules r;
  if (int rc = tc_rules(rules, vocab, &r)) return rc;
  const TcDraw d{draw->temperature, draw->top_k, draw->top_p, draw->min_p, draw->uniform};
  const int cols = ((vocab + kTcCluster - 1) / kTcCluster + 31) / 32 * 32;
  const int seg = (cols + kTcThreads - 1) / kTcThreads | 1;  // odd: a warp's threads are at different banks
  const bool vec = aligned(logits, 16) && stride * elem % 16 == 0;
  auto go = [&](auto kernel, auto* src) {
    if (!allow_smem(kernel, kTcHistBytes + kTcMaxLocal * 4)) return launch_result(cudaErrorInvalidValue);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)entries * kTcCluster);
    cfg.blockDim = dim3(kTcThreads);
    cfg.dynamicSmemBytes = kTcHistBytes + (size_t)cols * 4;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kTcCluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = take_chained_launch((cudaStream_t)stream) ? 2 : 1;
    return launch_result(cudaLaunchKernelEx(&cfg, kernel, src, (long long)stride, r, d, (int)vocab, cols, seg, append != 0, (long long*)tokens, logprobs, status));
  };
  if (elem == 4) return vec ? go(choose_tokens_kernel<float, true>, (const float*)logits) : go(choose_tokens_kernel<float, false>, (const float*)logits);
  return vec ? go(choose_tokens_kernel<uint16_t, true>, (const uint16_t*)logits) : go(choose_tokens_kernel<uint16_t, false>, (const uint16_t*)logits);
}
