// Layouts and arguments that the attention kernels (attention.hip) and their plan (attention_plan.hip) share.
#pragma once

#include "mlora_internal.h"

namespace mlora {

// A call's work is cut into tiles of packed rows: row r of a request and key head is (new token r / group, query head
// r % group of the key head's `group`), so the heads of a group share what is read of the cache.  Requests of up to FEW_ROWS rows
// (decoding ones) are one tile of the few-rows list, the others tiles of TALL_ROWS rows of the tall list.  A tile's span of the
// cache is cut into pieces where that evens out the work; a piece leaves its rows' sums, not yet divided, in a slot of the
// workspace; the last piece of a tile of few rows joins them, a launch of its own those of tall tiles.
//
// Few rows: spans above an even share of the whole are cut into equal pieces, a workgroup each.  Tall: the tiles stand in a line, each
// as long as its span and TALL_OVERHEAD tokens for its start and end; the line is cut into as many equal shares as the
// device holds workgroups, and a workgroup goes over the tiles of its share.  (One workgroup a piece: 616 of them for 512 places
// took a third longer.)  Where no tile can be long enough to be cut, each is a workgroup's: those of a request run side by side
// and find its K and V in the same L2 (16 prompts of 272 to 384 tokens 57.4 -> 55.1 us).
constexpr int FEW_ROWS = 16, TALL_ROWS = 128;
constexpr int AT_PIECE_STEP = 64;            // a piece's length is a multiple of this
constexpr int TALL_OVERHEAD = 192;

// plan buffer (int32 words): hdr[32] | few[max_few][8] | tall[max_tall][8] | joins[few_joins + tall_joins][8] | requests[n_req][8]
// | shares[max_shares + 1] | arrive[few_joins][kv_heads]
// record:  {request, first row, rows, begin, end, slot (-1: the tile's only piece), first new token in q, position of the
// request's new token 0}; the piece covers cache indices [begin, end); rows of the few-rows list hold the index of the tile's
// join in the upper half
// join:    {first slot, pieces, rows, first row, first new token in q, 0, 0, 0}; those of the few-rows list first, those of the tall
// list from few_joins on
// request: {blocks of WEIGHT_TOKENS cached tokens of the requests before, first new token in q, new tokens, cached tokens, tall tiles
// of the requests before, where its scores begin (two words), its row length of them}
// share:   its first record of the tall list
// arrive:  pieces of a tile that have left their sums, zero between calls
constexpr int AT_HDR = 32, AT_REC = 8;
enum AttnHdr { AH_FEW = 0, AH_TALL = 1, AH_TALL_JOINS = 2, AH_BLOCKS = 3, AH_SHARES = 4, AH_SCORES = 5 };
constexpr int WEIGHT_TOKENS = 256;
constexpr int64_t MAX_SCORES = 1 << 26;      // floats

struct AttnLayout {
  int64_t group;
  int64_t max_few, max_tall, max_shares;
  int few_joins, tall_joins;                 // room for joins of either list
  int64_t slots_few, slots_tall;
  int64_t scores;                            // room for scores of requests of few rows, floats
  int off_few, off_tall, off_joins, off_requests, off_shares, off_arrive;      // (words is checked to fit)
  int64_t words;
  int few_items;                             // (piece, key head) pairs the list is cut for
  bool few_whole;                            // as many requests with new tokens times key heads, or more: of like lengths, none is cut
  bool tall_each;                            // a share a tall tile: none is long enough to be cut
  int few_least, tall_least;                 // spans up to these are not cut
};

// A window as long as the longest cache bounds nothing; those that do, and the positions that a row's first token follows from, then
// stay within 2^30 either side of 0 (check_attention_plan), and their sums within 32 bits.
inline int window_of(const mlora_attention_plan &p) { return p.window >= p.max_kv_len ? 0 : p.window; }

AttnLayout attention_layout(const mlora_attention_plan &p);
int check_attention_plan(const mlora_attention_plan *p, const char *who);

// workspace: sums of the slots [slot][key head][rows][head_dim] floats, their references and
// sums [slot][key head][rows][4]; with weights the logarithm of each row's sum [token][query head], and where all of them fit
// (AH_SCORES) the scores of the requests of few rows [request][key head][row][token, from the first that any row sees on]
struct AttnWorkspace {
  int64_t few_o, tall_o, few_ml, tall_ml, lse, scores, bytes;
};
AttnWorkspace attention_workspace(const mlora_attention_plan &p, const AttnLayout &L, bool weights);

}  // namespace mlora
