// The plan of the attention calls of a batch: which rows of which request each workgroup takes, and which part of the
// request's cache.  Cut on the device from the lengths that are there, once per forward pass, for all its layers.
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

constexpr int AP_THREADS = 1024, AP_WAVES = AP_THREADS / 64;

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

// pieces of a span, none longer than `piece`; its length is evened out
__device__ __forceinline__ int cut(int len, int &piece) {
  if (len <= piece) return 1;
  const int k = (len + piece - 1) / piece;
  piece = ((len + k - 1) / k + AT_PIECE_STEP - 1) / AT_PIECE_STEP * AT_PIECE_STEP;
  return (len + piece - 1) / piece;
}

__device__ __forceinline__ int piece_length(int64_t total, int kv_heads, int items, int least) {
  const int64_t c = (total * kv_heads + items - 1) / items;
  const int64_t r = (c + AT_PIECE_STEP - 1) / AT_PIECE_STEP * AT_PIECE_STEP;
  return (int)(r < least ? least : r > (1 << 30) ? (1 << 30) : r);
}

// One workgroup; a thread owns a run of requests, so places in the lists follow from one sum over the threads.
__global__ __launch_bounds__(AP_THREADS) void attention_plan_kernel(PlanArgs a) {
  enum { FEW, TALL, JOINS, SLOTS_F, SLOTS_T, BLOCKS, COUNTS };
  __shared__ int64_t totals[2][AP_WAVES];
  __shared__ int counts[COUNTS][AP_WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per = (a.n_req + AP_THREADS - 1) / AP_THREADS;
  const int lo = min(tid * per, a.n_req), hi = min(lo + per, a.n_req);

  for (int64_t i = tid; i < a.L.max_joins * a.kv_heads; i += AP_THREADS) a.plan[a.L.off_arrive + i] = 0;
  int64_t few = 0, tall = 0;
  for (int b = lo; b < hi; ++b) {
    const Request r = request(a, b);
    int begin, end;
    if (r.rows > FEW_ROWS) {
      for (int row = 0; row < r.rows; row += TALL_ROWS) {
        span(a, r, row, min(TALL_ROWS, r.rows - row), begin, end);
        tall += end - begin;
      }
    } else if (r.rows > 0) {
      span(a, r, 0, r.rows, begin, end);
      few += end - begin;
    }
  }
  few = wave_sum(few);
  tall = wave_sum(tall);
  if (lane == 0) {
    totals[0][wave] = few;
    totals[1][wave] = tall;
  }
  __syncthreads();
  few = tall = 0;
  for (int i = 0; i < AP_WAVES; ++i) {
    few += totals[0][i];
    tall += totals[1][i];
  }
  const int few_piece = piece_length(few, a.kv_heads, a.L.few_items, a.L.few_least);
  const int tall_piece = piece_length(tall, a.kv_heads, a.L.tall_items, a.L.tall_least);

  int mine[COUNTS] = {0, 0, 0, 0, 0, 0};
  auto count = [&](int list, int slots, int len, int piece) {
    const int k = cut(len, piece);
    mine[list] += k;
    if (k > 1) {
      ++mine[JOINS];
      mine[slots] += k;
    }
  };
  auto blocks = [&](const Request &r) {
    if (r.rows == 0) return 0;
    int begin, end;
    span(a, r, 0, r.rows, begin, end);
    return (end - begin + WEIGHT_TOKENS - 1) / WEIGHT_TOKENS;
  };
  for (int b = lo; b < hi; ++b) {
    const Request r = request(a, b);
    int begin, end;
    if (r.rows > FEW_ROWS) {
      for (int row = 0; row < r.rows; row += TALL_ROWS) {
        span(a, r, row, min(TALL_ROWS, r.rows - row), begin, end);
        count(TALL, SLOTS_T, end - begin, tall_piece);
      }
    } else if (r.rows > 0) {
      span(a, r, 0, r.rows, begin, end);
      count(FEW, SLOTS_F, end - begin, few_piece);
    }
    mine[BLOCKS] += blocks(r);
  }
  int at[COUNTS];
#pragma unroll
  for (int c = 0; c < COUNTS; ++c) {
    int v = mine[c];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(v, d);
      if (lane >= d) v += up;
    }
    at[c] = v - mine[c];
    if (lane == 63) counts[c][wave] = v;
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c < COUNTS; ++c)
    for (int i = 0; i < wave; ++i) at[c] += counts[c][i];
  if (tid == AP_THREADS - 1) {
    // (requests that overlap in q could ask for more than the lists hold: what is beyond is left out)
    a.plan[AH_FEW] = (int)min<int64_t>(at[FEW] + mine[FEW], a.L.max_few);
    a.plan[AH_TALL] = (int)min<int64_t>(at[TALL] + mine[TALL], a.L.max_tall);
    a.plan[AH_JOINS] = (int)min<int64_t>(at[JOINS] + mine[JOINS], a.L.max_joins);
    a.plan[AH_BLOCKS] = at[BLOCKS] + mine[BLOCKS];
    a.plan[a.L.off_requests + (int64_t)a.n_req * AT_REQ] = at[BLOCKS] + mine[BLOCKS];
  }

  auto emit = [&](int b, const Request &r, int row0, int rows, int list, int slots, int piece) {
    int begin, end;
    span(a, r, row0, rows, begin, end);
    const int k = cut(end - begin, piece);
    const bool is_tall = list == TALL;
    const int64_t max_records = is_tall ? a.L.max_tall : a.L.max_few, max_slots = is_tall ? a.L.slots_tall : a.L.slots_few;
    int32_t *records = a.plan + (is_tall ? a.L.off_tall : a.L.off_few);
    const bool fits = at[list] + k <= max_records && (k == 1 || (at[slots] + k <= max_slots && at[JOINS] < a.L.max_joins));
    for (int i = 0; i < k; ++i) {
      if (at[list] + i >= max_records) break;
      int32_t *rec = records + (int64_t)(at[list] + i) * AT_REC;
      const int p0 = begin + i * piece;
      rec[0] = b;
      rec[1] = row0;
      rec[2] = fits ? (is_tall || k == 1 ? rows : rows | at[JOINS] << 16) : 0;
      rec[3] = k > 1 ? p0 : begin;
      rec[4] = k > 1 ? min(p0 + piece, end) : end;
      rec[5] = k > 1 ? at[slots] + i : -1;
      rec[6] = r.start;
      rec[7] = r.kv - r.n;
    }
    if (k > 1) {
      if (at[JOINS] < a.L.max_joins) {
        int32_t *join = a.plan + a.L.off_joins + (int64_t)at[JOINS] * AT_REC;
        join[0] = at[slots];
        join[1] = fits ? k : 0;
        join[2] = rows;
        join[3] = row0;
        join[4] = r.start;
        join[5] = is_tall;
        join[6] = join[7] = 0;
      }
      ++at[JOINS];
      at[slots] += k;
    }
    at[list] += k;
  };
  for (int b = lo; b < hi; ++b) {
    const Request r = request(a, b);
    int32_t *rq = a.plan + a.L.off_requests + (int64_t)b * AT_REQ;
    rq[0] = at[BLOCKS];
    rq[1] = r.start;
    rq[2] = r.n;
    rq[3] = r.kv;
    at[BLOCKS] += blocks(r);
    if (r.rows > FEW_ROWS) {      // the last rows see most: first
      for (int row = (r.rows - 1) / TALL_ROWS * TALL_ROWS; row >= 0; row -= TALL_ROWS)
        emit(b, r, row, min(TALL_ROWS, r.rows - row), TALL, SLOTS_T, tall_piece);
    } else if (r.rows > 0) {
      emit(b, r, 0, r.rows, FEW, SLOTS_F, few_piece);
    }
  }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace

AttnLayout attention_layout(const mlora_attention_plan &p) {
  AttnLayout L{};
  L.group = p.q_heads / p.kv_heads;
  L.few_items = 1024;
  L.tall_items = 512;
  L.few_least = 128;
  L.tall_least = 512;
  const int64_t T = p.n_tokens, n = p.n_req < T ? p.n_req : T;      // requests with new tokens
  const bool tall = p.max_seq_len * L.group > FEW_ROWS;
  // sum of ceil(span / piece) <= tiles + sum of spans / piece, and a tile of k > 1 pieces has a span above (k - 1) pieces
  const int64_t few_more = ceil_div(L.few_items, p.kv_heads), tall_more = ceil_div(L.tall_items, p.kv_heads);
  const int64_t few_cut = ceil_div(p.max_kv_len, L.few_least), tall_cut = ceil_div(p.max_kv_len, L.tall_least);
  const auto least = [](int64_t a, int64_t b) { return a < b ? a : b; };
  L.max_few = least(n + few_more, n * (few_cut > 1 ? few_cut : 1));
  L.slots_few = few_cut > 1 ? least(2 * few_more, n * few_cut) : 0;
  const int64_t tiles = tall ? T * L.group / TALL_ROWS + n : 0;
  L.max_tall = tall ? least(tiles + tall_more, tiles * (tall_cut > 1 ? tall_cut : 1)) : 0;
  L.slots_tall = tall && tall_cut > 1 ? least(2 * tall_more, tiles * tall_cut) : 0;
  L.max_joins = L.slots_few / 2 + L.slots_tall / 2;
  L.off_few = AT_HDR;
  L.off_tall = L.off_few + L.max_few * AT_REC;
  L.off_joins = L.off_tall + L.max_tall * AT_REC;
  L.off_requests = L.off_joins + L.max_joins * AT_REC;
  L.off_arrive = L.off_requests + (p.n_req + 1) * AT_REQ;
  L.words = L.off_arrive + L.max_joins * p.kv_heads;
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
  if (p->n_req > (1 << 20) || p->q_heads > 1024 || p->n_tokens * p->q_heads > (1ll << 30) || p->max_kv_len > (1 << 30) ||
      p->max_seq_len > (1 << 30))
    return fail(MLORA_ERR_NO_KERNEL, "%s: n_req=%lld n_tokens=%lld max_kv_len=%lld too large", who, (long long)p->n_req,
                (long long)p->n_tokens, (long long)p->max_kv_len);
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
             (int)L.group, (int)plan->max_seq_len, (int)plan->max_kv_len, plan->kv_heads, plan->window};
  hipLaunchKernelGGL(attention_plan_kernel, dim3(1), dim3(AP_THREADS), 0, (hipStream_t)stream, a);
  return check_launch("attention_plan_kernel");
}

}  // extern "C"
