// Masked attention, forward (rules and layouts: masked_attention.h).
//
// A task is kWaves x 32 QB rows of one (batch, head), or, where a head has few queries and shares
// its keys, of all heads of one key head (rows r = head g, query i: r = g n_query + i); it runs over
// the key tiles in which any pair of its rows attends, found 64 tiles at a time by one ballot, in
// which each lane judges one tile.  K and V tiles come into LDS by DMA, row-major, double-buffered,
// one barrier per tile; V's columns are read by transposing LDS reads.
//
// Softmax: online, one reference maximum per row, moved (and the sums rescaled) only when a logit
// passes it by more than 8 bits; P is rounded to the inputs' type for P V as the products take it,
// sums and outputs are kept in fp32.
#include "masked_attention.h"

namespace vgo {
namespace masked {
namespace {

// What a launch adds to the problem.
template <typename T>
struct Forward {
  Args<T> a;
  T* out;
  float* lse;     // or null
  float* part_o;  // splits > 1: [splits, batch * virtual heads, rows, D] unnormalised sums
  float* part_ml; // and [.., rows, 2] their reference maxima (log2) and row sums
  int pack;       // heads per task (1, or heads / kv_heads)
  int rows;       // pack * n_query
  int row_blocks, splits, tiles, tasks;
};

// The key tiles of one task that its work-group (`wg`) and this wave (`w`) take part in.
template <typename T>
struct Walk {
  const Args<T>& a;
  Range wg, w;
  int b, limit, prefix, end, base, tile;
  uint64_t todo, mine, full, whole;  // of tiles base .. base + 63
  bool in_mine, in_full, in_whole;   // of `tile`

  __device__ __forceinline__ Walk(const Args<T>& args, const Range& group, const Range& wave, int batch, int begin,
                                  int last)
      : a(args), wg(group), w(wave), b(batch), end(last), base(begin - 64), tile(0), todo(0) {
    limit = key_limit(a, b);
    prefix = prefix_of(a, b);
    end = min(end, (limit + kTile - 1) / kTile);
  }
  __device__ __forceinline__ bool next() {
    while (todo == 0) {
      base += 64;
      if (base >= end) return false;
      const int t = base + lane_id();
      bool any = t < end, all_w = false, any_w = false, whole_t = false;
      if (any) {
        Range k{};
        if (a.key_doc) k = info_range(a.key_info[static_cast<int64_t>(b) * ((a.n_key + kTile - 1) / kTile) + t]);
        k.lo = t * kTile, k.hi = min(k.lo + kTile, limit) - 1;
        bool all;
        judge(a, wg, k, prefix, any, all);
        judge(a, w, k, prefix, any_w, all_w);
        const bool inside = k.lo + kTile <= limit;
        all_w = all_w && inside;
        whole_t = inside && (!a.key_doc || k.docs_whole);
      }
      todo = __ballot(any), mine = __ballot(any && any_w), full = __ballot(all_w), whole = __ballot(whole_t);
    }
    const int bit = __builtin_ctzll(todo);
    todo &= todo - 1;
    tile = base + bit;
    in_mine = mine >> bit & 1, in_full = full >> bit & 1, in_whole = whole >> bit & 1;
    return true;
  }
};

template <typename T, int D, int QB, int kWaves>
struct Layout {
  static constexpr int kRowsPerWave = 32 * QB, kRows = kRowsPerWave * kWaves;
  static constexpr int kTiles = 4 * Tile<T, D>::kBytes;  // K and V, two buffers
  static constexpr int kMass = kTiles, kDocs = kMass + 2 * kTile * 4, kRange = kDocs + 2 * kTile * 4;
  static constexpr int kDistances = kRange + kWaves * 16;
};

template <typename T, int D, int QB, int kWaves>
__global__ __launch_bounds__(64 * kWaves, kWaves == 1 || D * sizeof(T) > 256 ? 1 : 2) void forward_kernel(const Forward<T> f) {
  typedef Tile<T, D> TL;
  typedef Layout<T, D, QB, kWaves> LO;
  typedef typename Op<T>::op8 op8;
  extern __shared__ __align__(16) char lds[];
  const Args<T>& a = f.a;
  const int lane = lane_id(), l32 = lane & 31, h = lane >> 5;
  const int wave = kWaves == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  // Heads, then key splits, then row blocks from the last on (the longest first under a causal mask).
  int task = xcd_remap(blockIdx.x, f.tasks);
  const int block = f.row_blocks - 1 - task % f.row_blocks;
  task /= f.row_blocks;
  const int split = task % f.splits;
  task /= f.splits;
  const int vheads = a.heads / f.pack, vh = task % vheads, b = task / vheads;
  const int kvh = vh * f.pack / (a.heads / a.kv_heads);
  const int row0 = block * LO::kRows + wave * LO::kRowsPerWave;
  const int start = first_position(a, b);

  // The wave's rows: operands, positions, documents.
  op8 q[QB][TL::kSteps];
  int pos[QB], doc[QB], head[QB], index[QB];
  bool stored[QB];
  const float* distance[QB];
  float slope2[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int r = row0 + 32 * qb + l32, rc = min(r, f.rows - 1);
    const int g = f.pack == 1 ? 0 : rc / a.n_query;
    index[qb] = rc - g * a.n_query;
    head[qb] = vh * f.pack + g;
    stored[qb] = r < f.rows;
    pos[qb] = start + index[qb];
    doc[qb] = a.query_doc ? a.query_doc[static_cast<int64_t>(b) * a.n_query + index[qb]] : 0;
    slope2[qb] = a.slopes ? a.slopes[head[qb]] * kLog2e : 0.0f;
    distance[qb] = reinterpret_cast<const float*>(lds + LO::kDistances) + (f.pack == 1 ? 0 : g * (2 * a.buckets.reach + 1));
    const T* src = a.q + b * a.qs[0] + head[qb] * a.qs[1] + index[qb] * a.qs[2] + 8 * h;
#pragma unroll
    for (int t = 0; t < TL::kSteps; ++t) q[qb][t] = *reinterpret_cast<const op8*>(src + 16 * t);
  }
  // Positions of rows first .. first + n: contiguous within a head, everything across heads.
  const auto positions = [&](int first, int n, Range& r) {
    const int last = min(first + n, f.rows) - 1;
    first = min(first, f.rows - 1);
    const bool one = f.pack == 1 || first / a.n_query == last / a.n_query;
    r.lo = start + (one ? first % a.n_query : 0);
    r.hi = start + (one ? last % a.n_query : a.n_query - 1);
  };
  Range rw{}, rg{};
  positions(row0, LO::kRowsPerWave, rw);
  positions(block * LO::kRows, LO::kRows, rg);
  if (a.query_doc) {
    int lo = INT_MAX, hi = -1, bad = 0;
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
      if (stored[qb]) {
        if (doc[qb] >= 0) lo = min(lo, doc[qb]), hi = max(hi, doc[qb]);
        bad |= doc[qb] < 0;
      }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
      lo = min(lo, __shfl_xor(lo, off)), hi = max(hi, __shfl_xor(hi, off));
      bad |= __shfl_xor(bad, off);
    }
    rw.doc_lo = __builtin_amdgcn_readfirstlane(lo), rw.doc_hi = __builtin_amdgcn_readfirstlane(hi);
    rw.docs_whole = __builtin_amdgcn_readfirstlane(bad) == 0;
    if constexpr (kWaves > 1) {
      int* slot = reinterpret_cast<int*>(lds + LO::kRange);
      if (lane == 0) slot[4 * wave] = lo, slot[4 * wave + 1] = hi;
      __syncthreads();
      rg.doc_lo = INT_MAX, rg.doc_hi = -1;
#pragma unroll
      for (int i = 0; i < kWaves; ++i)
        rg.doc_lo = min(rg.doc_lo, __builtin_amdgcn_readfirstlane(slot[4 * i])),
        rg.doc_hi = max(rg.doc_hi, __builtin_amdgcn_readfirstlane(slot[4 * i + 1]));
      rg.docs_whole = false;
    } else {
      rg = rw;
    }
  }
  if (a.table)
    for (int g = 0; g < f.pack; ++g)
      fill_distances(a, reinterpret_cast<float*>(lds + LO::kDistances) + g * (2 * a.buckets.reach + 1), vh * f.pack + g,
                     64 * kWaves);

  float mref[QB], lsum[QB];
  f32x16 o[QB][TL::kCols];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    mref[qb] = -kInf, lsum[qb] = 0.0f;
#pragma unroll
    for (int dt = 0; dt < TL::kCols; ++dt) o[qb][dt] = f32x16{};
  }

  const T* kbase = a.k + b * a.ks[0] + kvh * a.ks[1];
  const T* vbase = a.v + b * a.vs[0] + kvh * a.vs[1];
  const int* kdocs = a.key_doc ? a.key_doc + static_cast<int64_t>(b) * a.n_key : nullptr;
  const uint32_t lds0 = lds_offset(lds);
  const int per_split = (f.tiles + f.splits - 1) / f.splits;
  Walk<T> walk(a, rg, rw, b, split * per_split, min(f.tiles, (split + 1) * per_split));
  const int limit = walk.limit;
  int last[QB];  // of the keys that lengths and the causal mask leave a row
#pragma unroll
  for (int qb = 0; qb < QB; ++qb)
    last[qb] = min(limit, a.causal ? max(pos[qb] + 1, walk.prefix) : INT_MAX) - 1;

  const auto load = [&](int buf) {
    const int k0 = walk.tile * kTile;
    const auto live = [&](int j) { return kdocs == nullptr || kdocs[j] >= 0; };
    stage<T, D, kWaves>(kbase, a.ks[2], k0, limit, walk.in_whole, lds0 + (2 * buf) * TL::kBytes, live);
    stage<T, D, kWaves>(vbase, a.vs[2], k0, limit, walk.in_whole, lds0 + (2 * buf + 1) * TL::kBytes, live);
    if (wave == 0) {
      const uint32_t j = min(k0 + lane, a.n_key - 1) * 4u;
      if (a.mass) lds_dma4(a.mass, j, lds0 + LO::kMass + buf * kTile * 4);
      if (kdocs) lds_dma4(kdocs, j, lds0 + LO::kDocs + buf * kTile * 4);
    }
  };

  bool more = walk.next();
  int buf = 0;
  if (more) load(0);
  while (more) {
    const int k0 = walk.tile * kTile;
    const bool mine = walk.in_mine, full = walk.in_full;
    more = walk.next();
    wait_vmem<0>();
    __syncthreads();
    if (more) load(buf ^ 1);
    if (mine) {
      const char* kt = lds + 2 * buf * TL::kBytes;
      const char* vt = kt + TL::kBytes;
      f32x16 s[QB][2];
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) s[qb][sub] = f32x16{};
#pragma unroll
        for (int t = 0; t < TL::kSteps; ++t) {
          const op8 ka = TL::rows_op(kt, 32 * sub, t);
#pragma unroll
          for (int qb = 0; qb < QB; ++qb) s[qb][sub] = Op<T>::mma(ka, q[qb][t], s[qb][sub]);
        }
      }
      float c = a.scale * kLog2e;  // from s to the exponents of 2
      const bool plain = full && !a.cap2 && !a.mass && !a.slopes && !a.table;
      if (!plain) {
        const float* mass = reinterpret_cast<const float*>(lds + LO::kMass) + buf * kTile;
        const int* tags = reinterpret_cast<const int*>(lds + LO::kDocs) + buf * kTile;
        // Whether the tile's distances all lie beyond the buckets' reach, and on which side.
        const bool behind = k0 + kTile - 1 - rw.lo <= -a.buckets.reach, ahead = k0 - rw.hi >= a.buckets.reach;
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
          const float far = a.table ? distance[qb][ahead ? 2 * a.buckets.reach : 0] : 0.0f;
#pragma unroll
          for (int sub = 0; sub < 2; ++sub) {
            f32x16& x = s[qb][sub];
            const int j0 = 32 * sub + 4 * h;  // key of register r: k0 + j0 + 8 (r / 4) + r % 4
            if (a.cap2) {
#pragma unroll
              for (int r = 0; r < 16; ++r) x[r] = cap_tanh<T>(x[r] * a.inv_cap) * a.cap2;
            } else {
#pragma unroll
              for (int r = 0; r < 16; ++r) x[r] *= c;
            }
            if (a.mass) {
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                const f32x4 m = *reinterpret_cast<const f32x4*>(mass + j0 + 8 * g);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[4 * g + e] = fmaf(m[e], kLog2e, x[4 * g + e]);
              }
            }
            if (a.slopes) {
              const float d0 = static_cast<float>(k0 + j0 - pos[qb]);
#pragma unroll
              for (int r = 0; r < 16; ++r)
                x[r] = fmaf(-slope2[qb], fabsf(d0 + static_cast<float>(8 * (r / 4) + r % 4)), x[r]);
            }
            if (a.table) {
              if (behind || ahead) {
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] += far;
              } else {
                const int d0 = k0 + j0 - pos[qb];
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                  const int d = max(-a.buckets.reach, min(a.buckets.reach, d0 + 8 * (r / 4) + r % 4));
                  x[r] += distance[qb][d + a.buckets.reach];
                }
              }
            }
            if (!full) {
              const int last_r = last[qb] - k0 - j0;  // keys past it do not attend
#pragma unroll
              for (int r = 0; r < 16; ++r) x[r] = 8 * (r / 4) + r % 4 <= last_r ? x[r] : -kInf;
              if (kdocs) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                  const i32x4 tag = *reinterpret_cast<const i32x4*>(tags + j0 + 8 * g);
#pragma unroll
                  for (int e = 0; e < 4; ++e) x[4 * g + e] = tag[e] == doc[qb] ? x[4 * g + e] : -kInf;
                }
              }
            }
          }
        }
        c = 1.0f;
      }
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        float top = s[qb][0][0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, s[qb][0][r]);
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[qb][1][r]);
        top = half_max(top) * c;
        if (__any(top > mref[qb] + 8.0f)) {
          const float m = fmaxf(mref[qb], top);
          const float alpha = m == -kInf ? 1.0f : __builtin_amdgcn_exp2f(mref[qb] - m);
          mref[qb] = m;
          lsum[qb] *= alpha;
#pragma unroll
          for (int dt = 0; dt < TL::kCols; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[qb][dt][r] *= alpha;
        }
        const float off = mref[qb] == -kInf ? 0.0f : -mref[qb];
        float sum = 0.0f;
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float p = __builtin_amdgcn_exp2f(fmaf(s[qb][sub][r], c, off));
            s[qb][sub][r] = p;
            sum += p;
          }
        lsum[qb] += sum;
      }
#pragma unroll
      for (int kc = 0; kc < 4; ++kc) {
        op8 p[QB];
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) p[qb] = as_op<T>(s[qb][kc >> 1], kc & 1);
#pragma unroll
        for (int dt = 0; dt < TL::kCols; ++dt) {
          const op8 va = TL::cols_op(vt, dt, kc);
#pragma unroll
          for (int qb = 0; qb < QB; ++qb) o[qb][dt] = Op<T>::mma(va, p[qb], o[qb][dt]);
        }
      }
    }
    buf ^= 1;
  }

#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    if (!stored[qb]) continue;
    const bool dead = a.query_doc && doc[qb] < 0;
    float l = half_sum(lsum[qb]);
    if (dead) l = 0.0f;
    if (f.splits > 1) {
      const int64_t row = (static_cast<int64_t>(split) * a.batch * vheads + b * vheads + vh) * f.rows + row0 +
                          32 * qb + l32;
      float* dst = f.part_o + row * D;
#pragma unroll
      for (int dt = 0; dt < TL::kCols; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<f32x4*>(dst + 32 * dt + 8 * g + 4 * h) =
              f32x4{o[qb][dt][4 * g], o[qb][dt][4 * g + 1], o[qb][dt][4 * g + 2], o[qb][dt][4 * g + 3]};
      if (h == 0) f.part_ml[2 * row] = l == 0.0f ? -kInf : mref[qb], f.part_ml[2 * row + 1] = l;
      continue;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T* dst = f.out + b * a.os[0] + head[qb] * a.os[1] + index[qb] * a.os[2];
#pragma unroll
    for (int dt = 0; dt < TL::kCols; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f32x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = l == 0.0f ? 0.0f : o[qb][dt][4 * g + e] * inv;
        store4(dst + 32 * dt + 8 * g + 4 * h, y);
      }
    if (f.lse && h == 0)
      f.lse[(static_cast<int64_t>(b) * a.heads + head[qb]) * a.n_query + index[qb]] =
          l == 0.0f ? kInf : mref[qb] + __builtin_amdgcn_logf(l);
  }
}

// Joins the splits' states of each row: D / 4 lanes a row.
template <typename T, int D>
__global__ __launch_bounds__(256) void join_kernel(const Forward<T> f) {
  const Args<T>& a = f.a;
  constexpr int kLanes = D / 4;
  const int vheads = a.heads / f.pack;
  const int64_t n = static_cast<int64_t>(a.batch) * vheads * f.rows;
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / kLanes;
  const int d = static_cast<int>(threadIdx.x) % kLanes * 4;
  if (row >= n) return;
  float m = -kInf;
  for (int s = 0; s < f.splits; ++s) m = fmaxf(m, f.part_ml[2 * (s * n + row)]);
  float l = 0.0f;
  f32x4 y{};
  for (int s = 0; s < f.splits; ++s) {
    const float ms = f.part_ml[2 * (s * n + row)], ls = f.part_ml[2 * (s * n + row) + 1];
    if (ls == 0.0f) continue;  // nothing attended there
    const float w = ms == m ? 1.0f : __builtin_amdgcn_exp2f(ms - m);
    l = fmaf(w, ls, l);
    const f32x4 x = *reinterpret_cast<const f32x4*>(f.part_o + (s * n + row) * D + d);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = fmaf(w, x[e], y[e]);
  }
  const int vh = static_cast<int>(row / f.rows), r = static_cast<int>(row % f.rows);
  const int b = vh / vheads, head = vh % vheads * f.pack + r / a.n_query, i = r % a.n_query;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] *= inv;
  store4(f.out + b * a.os[0] + head * a.os[1] + i * a.os[2] + d, y);
  if (f.lse && d == 0)
    f.lse[(static_cast<int64_t>(b) * a.heads + head) * a.n_query + i] =
        l == 0.0f ? kInf : m + __builtin_amdgcn_logf(l);
}

// One wave per tile.
__global__ __launch_bounds__(256) void doc_info_kernel(const int* docs, const int* lengths, int n, int batch,
                                                       int tiles, int2* info) {
  const int id = blockIdx.x * 4 + (threadIdx.x >> 6), lane = lane_id();
  if (id >= batch * tiles) return;
  const int b = id / tiles, j = id % tiles * kTile + lane;
  const int limit = lengths ? max(0, min(n, lengths[b])) : n;
  const int doc = j < limit ? docs[static_cast<int64_t>(b) * n + j] : -1;
  int lo = doc < 0 ? INT_MAX : doc, hi = doc < 0 ? -1 : doc;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) lo = min(lo, __shfl_xor(lo, off)), hi = max(hi, __shfl_xor(hi, off));
  const bool whole = __all(doc >= 0);
  if (lane == 0) info[id] = int2{whole ? lo : ~lo, hi};
}

// How a problem is cut into tasks.
struct Plan {
  int pack, rows, row_blocks, splits, tiles, waves, blocks;  // blocks: QB
  int64_t tasks;
};

Plan plan_of(const vgo_masked_attn* p, int dtype) {
  Plan r{};
  const int group = static_cast<int>(p->heads / p->kv_heads);
  const int reach = p->bucket_table && p->n_starts ? p->bucket_starts[p->n_starts - 1] : 1;
  const bool table_fits = !p->bucket_table || static_cast<int64_t>(group) * (2 * reach + 1) * 4 <= 32768;
  r.pack = p->n_query < 32 && table_fits ? group : 1;
  r.rows = static_cast<int>(r.pack * p->n_query);
  r.tiles = static_cast<int>(tiles_of(p->n_key));
  const int64_t vheads = p->batch * (p->heads / r.pack);
  const int64_t cus = device_cus();
  const auto count = [&](int rows) { return vheads * ((r.rows + rows - 1) / rows); };
  r.waves = 4, r.blocks = 2;
  if (dtype == VGO_F32 || p->head_dim == 128 || count(256) < cus) r.blocks = 1;
  if (r.blocks == 1 && count(128) < cus) r.waves = 1;
  const int rows = 32 * r.blocks * r.waves;
  r.row_blocks = (r.rows + rows - 1) / rows;
  const int64_t tasks = vheads * r.row_blocks;
  r.splits = 1;
  if (r.waves == 1 && tasks < 4 * cus)
    r.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((4 * cus + tasks - 1) / tasks, r.tiles)));
  r.tasks = tasks * r.splits;
  return r;
}

size_t align16(size_t n) { return (n + 15) & ~static_cast<size_t>(15); }

size_t forward_bytes(const vgo_masked_attn* p, const Plan& plan) {
  size_t n = info_bytes(p);
  if (plan.splits > 1) {
    const size_t rows = static_cast<size_t>(plan.splits) * p->batch * (p->heads / plan.pack) * plan.rows;
    n += align16(rows * p->head_dim * 4) + align16(rows * 8);
  }
  return n;
}

template <typename T, int D, int QB, int kWaves>
int launch(const Forward<T>& f, hipStream_t stream) {
  typedef Layout<T, D, QB, kWaves> LO;
  const size_t bytes = LO::kDistances + (f.a.table ? static_cast<size_t>(f.pack) * (2 * f.a.buckets.reach + 1) * 4 : 0);
  const auto kernel = forward_kernel<T, D, QB, kWaves>;
  if (bytes > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (e != hipSuccess) return fail(VGO_ELAUNCH, std::string("masked_attn: ") + hipGetErrorString(e));
  }
  hipLaunchKernelGGL(kernel, dim3(f.tasks), dim3(64 * kWaves), bytes, stream, f);
  return check_launch("masked_attn");
}

template <typename T, int D>
int run(const vgo_masked_attn* p, const Plan& plan, void* out, const int64_t out_stride[3], float* lse, char* ws,
        hipStream_t stream) {
  Forward<T> f{};
  f.a = make_args<T>(p);
  for (int i = 0; i < 3; ++i) f.a.os[i] = out_stride[i];
  f.out = static_cast<T*>(out), f.lse = lse;
  f.pack = plan.pack, f.rows = plan.rows, f.row_blocks = plan.row_blocks, f.splits = plan.splits;
  f.tiles = plan.tiles, f.tasks = static_cast<int>(plan.tasks);
  launch_info(f.a, ws, stream);
  const int64_t rows = p->batch * (p->heads / plan.pack) * plan.rows;
  if (plan.splits > 1) {
    f.part_o = reinterpret_cast<float*>(ws + info_bytes(p));
    f.part_ml = reinterpret_cast<float*>(ws + info_bytes(p) + align16(plan.splits * rows * p->head_dim * 4));
  }
  int status;
  if (plan.waves == 1)
    status = launch<T, D, 1, 1>(f, stream);
  else if constexpr (sizeof(T) == 2 && D == 64)
    status = plan.blocks == 2 ? launch<T, D, 2, 4>(f, stream) : launch<T, D, 1, 4>(f, stream);
  else
    status = launch<T, D, 1, 4>(f, stream);
  if (status != VGO_OK || plan.splits == 1) return status;
  const unsigned groups = static_cast<unsigned>((rows * (D / 4) + 255) / 256);
  hipLaunchKernelGGL((join_kernel<T, D>), dim3(groups), dim3(256), 0, stream, f);
  return check_launch("masked_attn join");
}

}  // namespace

void launch_doc_info(const int* docs, const int* lengths, int n, int batch, int tiles, int2* info,
                     hipStream_t stream) {
  hipLaunchKernelGGL(doc_info_kernel, dim3((batch * tiles + 3) / 4), dim3(256), 0, stream, docs, lengths, n, batch,
                     tiles, info);
}

size_t info_bytes(const vgo_masked_attn* p) {
  return p->key_documents ? align16(static_cast<size_t>(p->batch) * (tiles_of(p->n_key) + tiles_of(p->n_query)) * 8)
                          : 0;
}

bool strides_fit(const int64_t stride[3], int64_t head_dim, int dtype) {
  const int64_t size = dtype == VGO_F32 ? 4 : 2;
  for (int i = 0; i < 3; ++i)
    if (stride[i] < 0 || stride[i] * size % 16 != 0) return false;
  return stride[2] * size * kTile < (int64_t{1} << 31);  // 32-bit offsets within a tile
}

int check_buckets(int64_t count, const int32_t* starts, int n_starts, int bidirectional) {
  VGO_REQUIRE(n_starts >= 0 && n_starts <= kMaxStarts && (n_starts == 0 || starts), "buckets: at most 128 starts");
  VGO_REQUIRE(count >= (bidirectional ? 2 : 1) * (n_starts + 1) && count <= 4096 && (!bidirectional || count % 2 == 0),
              "buckets: the table must hold every bucket, and at most 4096");
  for (int t = 0; t < n_starts; ++t)
    VGO_REQUIRE(starts[t] >= 1 && starts[t] <= 1024 && (t == 0 || starts[t] >= starts[t - 1]),
                "buckets: starts must ascend within 1 .. 1024");
  return VGO_OK;
}

int check_problem(const vgo_masked_attn* p, int dtype) {
  VGO_REQUIRE(p, "masked_attn: null problem");
  VGO_REQUIRE(dtype == VGO_F32 || dtype == VGO_BF16 || dtype == VGO_F16, "masked_attn: unsupported dtype");
  VGO_REQUIRE(p->head_dim == 64 || p->head_dim == 128, "masked_attn: head_dim must be 64 or 128");
  VGO_REQUIRE(p->batch >= 0 && p->heads >= 1 && p->kv_heads >= 1 && p->n_query >= 0 && p->n_key >= 0,
              "masked_attn: negative size");
  VGO_REQUIRE(p->heads % p->kv_heads == 0, "masked_attn: heads must be a multiple of the key heads");
  const int64_t most = int64_t{1} << 28;
  VGO_REQUIRE(p->n_query < most && p->n_key < most && p->batch < most && p->heads < most,
              "masked_attn: sizes are below 2^28");
  // Task counts, and rows of all heads, are 32-bit.
  VGO_REQUIRE(p->batch * p->heads < most && (p->batch * p->heads) * (p->n_query / 32 + 1) < most &&
                  p->batch * (p->heads / p->kv_heads) * 32 < most,
              "masked_attn: too many rows");
  VGO_REQUIRE(p->scale > 0.0f && p->scale < kInf, "masked_attn: the scale must be positive and finite");
  VGO_REQUIRE(p->score_cap >= 0.0f && p->score_cap < kInf, "masked_attn: the score cap must be finite and not negative");
  VGO_REQUIRE(!p->prefix_lengths || p->causal, "masked_attn: a prefix goes with a causal mask");
  VGO_REQUIRE(!p->query_documents == !p->key_documents, "masked_attn: documents of queries and keys go together");
  if (p->bucket_table) {
    const int status = check_buckets(p->n_buckets, p->bucket_starts, p->n_starts, p->bidirectional);
    if (status != VGO_OK) return status;
  }
  if (p->batch == 0 || p->n_query == 0) return VGO_OK;
  VGO_REQUIRE(p->q && aligned(p->q, 16) && strides_fit(p->q_stride, p->head_dim, dtype),
              "masked_attn: q must be 16-byte aligned, with strides of whole 16 bytes");
  if (p->n_key == 0) return VGO_OK;
  VGO_REQUIRE(p->k && p->v && aligned(p->k, 16) && aligned(p->v, 16) &&
                  strides_fit(p->k_stride, p->head_dim, dtype) && strides_fit(p->v_stride, p->head_dim, dtype),
              "masked_attn: k and v must be 16-byte aligned, with strides of whole 16 bytes");
  return VGO_OK;
}

}  // namespace masked
}  // namespace vgo

extern "C" int vgo_masked_attn_workspace(const vgo_masked_attn* problem, int dtype, size_t* bytes) {
  using namespace vgo;
  using namespace vgo::masked;
  const int status = check_problem(problem, dtype);
  if (status != VGO_OK) return status;
  VGO_REQUIRE(bytes, "masked_attn: null pointer");
  *bytes = problem->batch == 0 || problem->n_query == 0 ? 0 : forward_bytes(problem, plan_of(problem, dtype));
  return VGO_OK;
}

extern "C" int vgo_masked_attn_fwd(const vgo_masked_attn* problem, void* out, const int64_t out_stride[3], float* lse,
                                   int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace vgo;
  using namespace vgo::masked;
  const int status = check_problem(problem, dtype);
  if (status != VGO_OK) return status;
  if (problem->batch == 0 || problem->n_query == 0) return VGO_OK;
  VGO_REQUIRE(out && out_stride && aligned(out, 16) && strides_fit(out_stride, problem->head_dim, dtype),
              "masked_attn: out must be 16-byte aligned, with strides of whole 16 bytes");
  const Plan plan = plan_of(problem, dtype);
  const size_t need = forward_bytes(problem, plan);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(VGO_EWORKSPACE, "masked_attn: workspace of " + std::to_string(need) + " bytes needed");
  char* ws = static_cast<char*>(workspace);
  const bool wide = problem->head_dim == 128;
  const hipStream_t s = as_stream(stream);
  switch (dtype) {
    case VGO_BF16:
      return wide ? run<bf16_t, 128>(problem, plan, out, out_stride, lse, ws, s)
                  : run<bf16_t, 64>(problem, plan, out, out_stride, lse, ws, s);
    case VGO_F16:
      return wide ? run<f16_t, 128>(problem, plan, out, out_stride, lse, ws, s)
                  : run<f16_t, 64>(problem, plan, out, out_stride, lse, ws, s);
    default:
      return wide ? run<float, 128>(problem, plan, out, out_stride, lse, ws, s)
                  : run<float, 64>(problem, plan, out, out_stride, lse, ws, s);
  }
}
