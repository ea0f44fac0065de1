// The plan of the attention calls of a batch: which rows of which request each workgroup takes, and which part of the
// request's cache.  Cut on the device from the lengths that are there, once per forward pass, for all its layers.
//
// One workgroup: requests, then tall tiles, a thread each, with a running sum over the threads for where each one's records go.
// Bound by the latency of its passes (8 us for 256 decoding requests, 15 for 130 mixed ones).
#include "attention.h"
#include "kernel_common.h"

namespace mlora {

namespace {

struct PlanArgs {
  int32_t *plan;
  const int32_t *start, *seq, *kv;
  AttnLayout L;
  int64_t n_tokens;
  int n_req, group, max_seq, max_kv, kv_heads, window;
};

constexpr int AP_THREADS = 512, AP_WAVES = AP_THREADS / 64;

struct Request {
  int n, start, kv, rows;
};

// Requests with nothing new, and those whose lengths the call's tensors do not hold, have no rows.
__device__ __forceinline__ Request request(const PlanArgs &a, int b) {
  Request r{a.seq[b], a.start[b], a.kv[b], 0};
  r.kv = min(max(r.kv, 0), a.max_kv);
  if (r.n < 1 || r.n > a.max_seq || r.start < 0 || (int64_t)r.start + r.n > a.n_tokens) r.n = 0;
  r.rows = r.n * a.group;
  return r;
}

// What rows [row0, row0 + rows) of a request see of its cache: [begin, end)
__device__ __forceinline__ void span(const PlanArgs &a, const Request &r, int row0, int rows, int &begin, int &end) {
  const int64_t pos0 = (int64_t)r.kv - r.n;
  const int64_t first = pos0 + row0 / a.group, last = pos0 + (row0 + rows - 1) / a.group;
  begin = a.window > 0 && first + 1 > a.window ? (int)(first + 1 - a.window) : 0;
  end = (int)(last + 1 > 0 ? last + 1 : 0);
  if (begin > end) begin = end;
}

__device__ __forceinline__ int64_t wave_sum(int64_t v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  return v;
}

// Sum over the workgroup, for everyone
__device__ __forceinline__ int64_t block_sum(int64_t v, int64_t (&part)[AP_WAVES]) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
  for (int i = 0; i < AP_WAVES; ++i) v += part[i];
  return v;
}

// Sum over the threads before this one, and over all in `total`
__device__ __forceinline__ int64_t block_before(int64_t mine, int64_t &total, int64_t (&part)[AP_WAVES]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t v = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t up = __shfl_up(v, d);
    if (lane >= d) v += up;
  }
  __syncthreads();
  if (lane == 63) part[wave] = v;
  __syncthreads();
  int64_t before = v - mine;
  total = 0;
  for (int i = 0; i < AP_WAVES; ++i) {
    before += i < wave ? part[i] : 0;
    total += part[i];
  }
  return before;
}

// pieces of a span, none longer than `piece`; its length is evened out
__device__ __forceinline__ int cut(int len, int &piece) {
  if (len <= piece) return 1;
  const int k = (len + piece - 1) / piece;
  piece = ((len + k - 1) / k + AT_PIECE_STEP - 1) / AT_PIECE_STEP * AT_PIECE_STEP;
  return (len + piece - 1) / piece;
}

// counts of records, slots and joins travel through the sums as one number (each below 2^20: csrc/attention_plan.hip, layout)
__device__ __forceinline__ int64_t pack(int64_t records, int64_t slots, int64_t joins) { return records | slots << 21 | joins << 42; }
constexpr int64_t PACKED = (1 << 21) - 1;

// One workgroup, a thread per request and then per tall tile, in rounds where there are more.
// EACH: the layout's tall_each
template <bool EACH>
__global__ __launch_bounds__(AP_THREADS) void attention_plan_kernel(PlanArgs a) {
  __shared__ int64_t part[AP_WAVES];
  const int tid = threadIdx.x;
  int32_t *requests = a.plan + a.L.off_requests, *shares = a.plan + a.L.off_shares;
  for (int64_t i = tid; i < (int64_t)a.L.few_joins * a.kv_heads; i += AP_THREADS) a.plan[a.L.off_arrive + i] = 0;

  // ---- requests
  int64_t few = 0, blocks_before = 0, tiles = 0, scores = 0;
  for (int b0 = 0; b0 < a.n_req; b0 += AP_THREADS) {
    const int b = b0 + tid;
    Request r{};
    int begin = 0, end = 0, n_blocks = 0, n_tiles = 0, row_scores = 0;
    int64_t n_scores = 0;
    if (b < a.n_req) {
      r = request(a, b);
      if (r.rows > 0) {
        span(a, r, 0, r.rows, begin, end);
        n_blocks = (end - begin + WEIGHT_TOKENS - 1) / WEIGHT_TOKENS;
        n_tiles = r.rows > FEW_ROWS ? (r.rows + TALL_ROWS - 1) / TALL_ROWS : 0;
        if (n_tiles == 0) {
          few += end - begin;
          row_scores = (end - begin + 63) / 64 * 64;
          n_scores = (int64_t)r.rows * a.kv_heads * row_scores;
        }
      }
    }
    int64_t all, all_scores;
    const int64_t before = block_before(n_blocks | (int64_t)n_tiles << 32, all, part);
    const int64_t its_scores = scores + block_before(n_scores, all_scores, part);
    if (b < a.n_req) {
      int32_t *rq = requests + (int64_t)b * AT_REC;
      rq[0] = (int32_t)(blocks_before + (before & 0xffffffff));
      rq[1] = r.start;
      rq[2] = r.n;
      rq[3] = r.kv;
      rq[4] = (int32_t)(tiles + (before >> 32));
      rq[5] = (int32_t)its_scores;
      rq[6] = (int32_t)(its_scores >> 32);
      rq[7] = row_scores;
    }
    blocks_before += all & 0xffffffff;
    tiles += all >> 32;
    scores += all_scores;
  }
  if (tid == 0) {
    a.plan[AH_BLOCKS] = (int32_t)blocks_before;
    a.plan[AH_SCORES] = scores <= a.L.scores;
  }
  few = block_sum(few, part);
  int64_t records = 0, slots = 0, joins = 0;

  auto emit_join = [&](int64_t at, int64_t first, int64_t max, int64_t slot0, int pieces, int rows, int row0, int start) {
    if (at >= max) return;
    int32_t *j = a.plan + a.L.off_joins + (first + at) * AT_REC;
    j[0] = (int32_t)slot0;
    j[1] = pieces;
    j[2] = rows;
    j[3] = row0;
    j[4] = start;
    j[5] = j[6] = j[7] = 0;
  };
  auto emit = [&](int32_t *list, int64_t at, int64_t max, int b, int row0, int rows, int begin, int end, int64_t slot, const Request &r) {
    if (at >= max) return;
    int32_t *rec = list + at * AT_REC;
    rec[0] = b;
    rec[1] = row0;
    rec[2] = rows;
    rec[3] = begin;
    rec[4] = end;
    rec[5] = (int32_t)slot;
    rec[6] = r.start;
    rec[7] = r.kv - r.n;
  };

  // ---- few rows: a request's tile into equal pieces
  const int64_t even = ((few * a.kv_heads + a.L.few_items - 1) / a.L.few_items + AT_PIECE_STEP - 1) / AT_PIECE_STEP * AT_PIECE_STEP;
  const int few_piece = (int)(even < a.L.few_least ? a.L.few_least : even > (1 << 30) ? (1 << 30) : even);
  for (int b0 = 0; b0 < a.n_req; b0 += AP_THREADS) {
    const int b = b0 + tid;
    Request r{};
    int begin = 0, end = 0, k = 0, piece = few_piece;
    if (b < a.n_req) {
      r = request(a, b);
      if (r.rows > 0 && r.rows <= FEW_ROWS) {
        span(a, r, 0, r.rows, begin, end);
        k = cut(end - begin, piece);
      }
    }
    int64_t all;
    const int64_t before = block_before(k > 0 ? pack(k, k > 1 ? k : 0, k > 1) : 0, all, part);
    const int64_t rec = records + (before & PACKED), slot = slots + (before >> 21 & PACKED), join = joins + (before >> 42);
    // (requests that overlap in q could ask for more than the lists hold: what is beyond is left out)
    const bool fits = rec + k <= a.L.max_few && (k < 2 || (slot + k <= a.L.slots_few && join < a.L.few_joins));
    for (int i = 0; i < k; ++i)
      emit(a.plan + a.L.off_few, rec + i, a.L.max_few, b, 0, !fits ? 0 : k > 1 ? r.rows | (int)join << 16 : r.rows, begin + (k > 1 ? i * piece : 0),
           k > 1 ? min(begin + (i + 1) * piece, end) : end, k > 1 ? slot + i : -1, r);
    if (k > 1) emit_join(join, 0, a.L.few_joins, slot, fits ? k : 0, r.rows, 0, r.start);
    records += all & PACKED;
    slots += all >> 21 & PACKED;
    joins += all >> 42;
  }
  if (tid == 0) a.plan[AH_FEW] = (int)min<int64_t>(records, a.L.max_few);

  auto finish = [&](int64_t tall, int64_t tall_joins, int64_t n_shares) {
    if (tid != 0) return;
    tall = min<int64_t>(tall, a.L.max_tall);
    a.plan[AH_TALL] = (int32_t)tall;
    a.plan[AH_TALL_JOINS] = (int32_t)min<int64_t>(tall_joins, a.L.tall_joins);
    a.plan[AH_SHARES] = (int32_t)n_shares;
    shares[n_shares] = (int32_t)tall;
  };

  // ---- tall tiles, in a line
  struct Place {
    Request r;
    int b, row0, rows, begin, end;
  };
  auto tile = [&](int64_t t) {
    // the last request whose tiles begin at or before t
    int lo = 0, hi = a.n_req;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (requests[(int64_t)mid * AT_REC + 4] <= t) lo = mid;
      else hi = mid;
    }
    const int32_t *rq = requests + (int64_t)lo * AT_REC;
    Place p;
    p.r = Request{rq[2], rq[1], rq[3], rq[2] * a.group};
    p.b = lo;
    p.row0 = (int)((t - rq[4]) * TALL_ROWS);
    p.rows = min(TALL_ROWS, p.r.rows - p.row0);
    span(a, p.r, p.row0, p.rows, p.begin, p.end);
    return p;
  };
  __syncthreads();                       // (the requests are written)
  if constexpr (EACH) {
    const int64_t n = min(min(tiles, a.L.max_tall), a.L.max_shares);
    for (int64_t t = tid; t < n; t += AP_THREADS) {
      const Place p = tile(t);
      emit(a.plan + a.L.off_tall, t, a.L.max_tall, p.b, p.row0, p.rows, p.begin, p.end, -1, p.r);
      shares[t] = (int32_t)t;
    }
    finish(n, 0, n);
    return;
  }
  int64_t line = 0;
  for (int64_t t = tid; t < tiles; t += AP_THREADS) {
    const Place p = tile(t);
    line += p.end - p.begin + TALL_OVERHEAD;
  }
  line = block_sum(line, part);
  int n_shares = (int)min<int64_t>((line + a.L.tall_least - 1) / a.L.tall_least, a.L.max_shares);
  const int64_t share = n_shares > 0 ? (line + n_shares - 1) / n_shares : 1;
  n_shares = (int)((line + share - 1) / share);      // (one that begins behind the line is none)
  records = slots = joins = 0;
  int64_t at = 0;                        // where on the line the round's first tile begins
  for (int64_t t0 = 0; t0 < tiles; t0 += AP_THREADS) {
    const int64_t t = t0 + tid;
    Place p{};
    int64_t length = 0;
    if (t < tiles) {
      p = tile(t);
      length = p.end - p.begin + TALL_OVERHEAD;
    }
    int64_t all;
    const int64_t from = at + block_before(length, all, part);
    at += all;
    // f(index of the share that begins here, cut) for the shares that begin within the tile; a cut near an end is none
    auto cuts = [&](auto f) {
      const int len = p.end - p.begin;
      int64_t step = share;
      asm volatile("" : "+v"(step));     // (as a vector: the scalars of the division would be spilled)
      for (int64_t j = (from + step - 1) / step; j * step < from + length; ++j) {
        const int64_t inside = j * step - from - TALL_OVERHEAD / 2;
        int cut = (int)((inside + AT_PIECE_STEP / 2) / AT_PIECE_STEP * AT_PIECE_STEP);
        if (inside < a.L.tall_least / 2 || len < a.L.tall_least) cut = inside * 2 < len ? 0 : len;
        else if (inside > len - a.L.tall_least / 2) cut = len;
        f(j, cut);
      }
    };
    int k = 0;
    if (t < tiles) {
      int last = 0;
      const int len = p.end - p.begin;
      cuts([&](int64_t, int cut) {
        if (cut > last && cut < len) {
          ++k;
          last = cut;
        }
      });
      ++k;
    }
    const int64_t before = block_before(k > 0 ? pack(k, k > 1 ? k : 0, k > 1) : 0, all, part);
    const int64_t rec = records + (before & PACKED), slot = slots + (before >> 21 & PACKED), join = joins + (before >> 42);
    if (t < tiles) {
      const bool fits = rec + k <= a.L.max_tall && (k < 2 || (slot + k <= a.L.slots_tall && join < a.L.tall_joins));
      const int len = p.end - p.begin;
      int last = 0, i = 0;
      cuts([&](int64_t j, int cut) {
        if (cut > last && cut < len) {
          emit(a.plan + a.L.off_tall, rec + i, a.L.max_tall, p.b, p.row0, fits ? p.rows : 0, p.begin + last, p.begin + cut, slot + i, p.r);
          ++i;
          last = cut;
        }
        // (the tile's last piece begins a share that is cut at the tile's start or within it; one cut at its end begins with the next tile)
        if (j < n_shares) shares[j] = (int32_t)(rec + (cut >= len && len > 0 ? k : i));
      });
      emit(a.plan + a.L.off_tall, rec + i, a.L.max_tall, p.b, p.row0, fits ? p.rows : 0, p.begin + last, p.end, k > 1 ? slot + i : -1, p.r);
      if (k > 1) emit_join(join, a.L.few_joins, a.L.tall_joins, slot, fits ? k : 0, p.rows, p.row0, p.r.start);
    }
    records += all & PACKED;
    slots += all >> 21 & PACKED;
    joins += all >> 42;
  }
  finish(records, joins, n_shares);
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace

AttnLayout attention_layout(const mlora_attention_plan &p) {
  AttnLayout L{};
  L.group = p.q_heads / p.kv_heads;
  L.few_items = 1024;
  L.few_least = 128;
  L.tall_least = 512;
  constexpr int64_t TALL_PLACES = 512;       // two workgroups on each of 256 CUs
  const int64_t T = p.n_tokens, n = p.n_req < T ? p.n_req : T;      // requests with new tokens
  const bool tall = p.max_seq_len * L.group > FEW_ROWS;
  const auto least = [](int64_t a, int64_t b) { return a < b ? a : b; };
  // few rows: sum of ceil(span / piece) <= tiles + sum of spans / piece, and a tile of k > 1 pieces has a span above (k - 1) pieces
  const int64_t few_more = ceil_div(L.few_items, p.kv_heads), few_cut = ceil_div(p.max_kv_len, L.few_least);
  L.max_few = least(n + few_more, n * (few_cut > 1 ? few_cut : 1));
  L.slots_few = few_cut > 1 ? least(2 * few_more, n * few_cut) : 0;
  // tall: a share's beginning cuts one tile at most; k pieces of a tile are k - 1 cuts, and a cut tile has two pieces at least
  const int64_t tiles = tall ? T * L.group / TALL_ROWS + n : 0;
  L.tall_each = p.max_kv_len < L.tall_least;
  L.max_shares = least(TALL_PLACES / p.kv_heads > 0 ? TALL_PLACES / p.kv_heads : 1, tiles * ceil_div(p.max_kv_len + TALL_OVERHEAD, L.tall_least));
  if (L.tall_each) L.max_shares = tiles;
  L.max_tall = tiles > 0 ? tiles + (p.max_kv_len >= L.tall_least ? L.max_shares : 0) : 0;
  L.slots_tall = tiles > 0 && p.max_kv_len >= L.tall_least ? 2 * L.max_shares : 0;
  L.few_joins = (int)(L.slots_few / 2);
  L.tall_joins = (int)(L.slots_tall / 2);
  const int64_t rows = least(FEW_ROWS, p.max_seq_len * L.group);
  L.scores = least(MAX_SCORES, n * least(MAX_SCORES, rows * p.kv_heads * ceil_div(p.max_kv_len, 64) * 64));
  int64_t at = AT_HDR;
  auto take = [&](int64_t words) {
    const int64_t here = at;
    at += words;
    return (int)here;
  };
  L.off_few = take(L.max_few * AT_REC);
  L.off_tall = take(L.max_tall * AT_REC);
  L.off_joins = take(((int64_t)L.few_joins + L.tall_joins) * AT_REC);
  L.off_requests = take(p.n_req * AT_REC);
  L.off_shares = take(L.max_shares + 1);
  L.off_arrive = take((int64_t)L.few_joins * p.kv_heads);
  L.words = at;
  return L;
}

AttnWorkspace attention_workspace(const mlora_attention_plan &p, const AttnLayout &L, bool weights) {
  AttnWorkspace w{};
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += align_up(bytes, 256);
    return here;
  };
  w.few_o = take(L.slots_few * p.kv_heads * FEW_ROWS * p.head_dim * 4);
  w.tall_o = take(L.slots_tall * p.kv_heads * TALL_ROWS * p.head_dim * 4);
  w.few_ml = take(L.slots_few * p.kv_heads * FEW_ROWS * 16);
  w.tall_ml = take(L.slots_tall * p.kv_heads * TALL_ROWS * 16);
  w.lse = take(weights ? p.n_tokens * p.q_heads * 4 : 0);
  w.scores = take(weights ? L.scores * 4 : 0);
  w.bytes = at;
  return w;
}

int check_attention_plan(const mlora_attention_plan *p, const char *who) {
  if (!p) return fail(MLORA_ERR_INVALID, "%s: plan is null", who);
  if (p->n_req < 0 || p->n_tokens < 0 || p->max_seq_len < 0 || p->max_kv_len < 0 || p->window < 0)
    return fail(MLORA_ERR_INVALID, "%s: negative size", who);
  if (p->q_heads < 1 || p->kv_heads < 1 || p->q_heads % p->kv_heads)
    return fail(MLORA_ERR_INVALID, "%s: q_heads=%d is not a multiple of kv_heads=%d", who, p->q_heads, p->kv_heads);
  const int d = p->head_dim;
  if (d != 32 && d != 64 && d != 96 && d != 128 && d != 256)
    return fail(MLORA_ERR_NO_KERNEL, "No suitable kernel. %s: head_dim=%d (32, 64, 96, 128 or 256)", who, d);
  if (p->page_size < 1 || p->page_size > 256 || (p->page_size & (p->page_size - 1)))
    return fail(MLORA_ERR_NO_KERNEL, "No suitable kernel. %s: page_size=%d (a power of two up to 256)", who, p->page_size);
  // rows, cache indices and positions are kept in 32 bits
  if (p->n_req > (1 << 20) || p->q_heads > 1024 || p->n_tokens > (1 << 30) || p->n_tokens * p->q_heads > (1 << 30) || p->max_kv_len > (1 << 30) ||
      p->max_seq_len > (1 << 30))
    return fail(MLORA_ERR_NO_KERNEL, "%s: n_req=%lld n_tokens=%lld max_kv_len=%lld too large", who, (long long)p->n_req,
                (long long)p->n_tokens, (long long)p->max_kv_len);
  if (p->n_req * ((p->max_kv_len + WEIGHT_TOKENS - 1) / WEIGHT_TOKENS) > 0x7fffffff)
    return fail(MLORA_ERR_NO_KERNEL, "%s: n_req=%lld times max_kv_len=%lld too large", who, (long long)p->n_req, (long long)p->max_kv_len);
  if (attention_layout(*p).words > 0x7fffffff) return fail(MLORA_ERR_NO_KERNEL, "%s: the plan would have more than 2^31 - 1 words", who);
  return MLORA_OK;
}

}  // namespace mlora

using namespace mlora;

extern "C" {

size_t mlora_attention_plan_bytes(const mlora_attention_plan *plan) {
  return check_attention_plan(plan, "attention_plan_bytes") ? 0 : (size_t)attention_layout(*plan).words * 4;
}

size_t mlora_attention_workspace_bytes(const mlora_attention_plan *plan, int32_t weights) {
  if (check_attention_plan(plan, "attention_workspace_bytes")) return 0;
  return (size_t)attention_workspace(*plan, attention_layout(*plan), weights != 0).bytes;
}

int mlora_build_attention_plan(void *stream, const mlora_attention_plan *plan, const int32_t *b_start_loc,
                               const int32_t *b_seq_len, const int32_t *b_kv_len) {
  if (int rc = check_attention_plan(plan, "build_attention_plan")) return rc;
  const AttnLayout L = attention_layout(*plan);
  if (!plan->dev || plan->bytes < (size_t)L.words * 4 || (reinterpret_cast<uintptr_t>(plan->dev) & 15))
    return fail(MLORA_ERR_WORKSPACE, "build_attention_plan: plan buffer has %zu bytes (16-byte aligned), needs %lld", plan->dev ? plan->bytes : 0,
                (long long)L.words * 4);
  if (plan->n_req > 0 && (!b_start_loc || !b_seq_len || !b_kv_len))
    return fail(MLORA_ERR_INVALID, "build_attention_plan: null pointer");
  PlanArgs a{static_cast<int32_t *>(plan->dev), b_start_loc, b_seq_len, b_kv_len, L, plan->n_tokens, (int)plan->n_req,
             (int)L.group, (int)plan->max_seq_len, (int)plan->max_kv_len, plan->kv_heads, window_of(*plan)};
  hipLaunchKernelGGL(L.tall_each ? attention_plan_kernel<true> : attention_plan_kernel<false>, dim3(1), dim3(AP_THREADS), 0, (hipStream_t)stream, a);
  return check_launch("attention_plan_kernel");
}

}  // extern "C"
