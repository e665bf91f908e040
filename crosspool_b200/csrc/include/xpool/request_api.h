/* Operators of a batch whose requests share a prompt prefix, bring low-rank adapters of their own and put controls on their
 * logits (shared_prefix.cu, lora.cu, logit_controls.cu). Functions return 0, or a negative code when the arguments are outside
 * what the kernels cover (nothing was launched then) or a launch failed (-100 - cudaError_t). */
#ifndef XPOOL_REQUEST_API_H_
#define XPOOL_REQUEST_API_H_

#include <stdint.h>

#include "xpool/api.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Decode attention of rows that share prefixes. A piece is a range of a prefix and the consecutive rows that read it together;
 * every piece of a row leaves a partial result, to which the row's own tokens are added. */
typedef struct XpPrefixPiece {
  int leader;                 /* row whose block table names the prefix's pages */
  int row0, rows;             /* rows of the piece */
  int tok0, tok1;             /* tokens [tok0, tok1) of the sequence, tok0 a multiple of 128, tok1 of 16 */
  int part;                   /* index of the partial result of these rows */
  int pad0, pad1;
} XpPrefixPiece;

typedef struct XpDecodeSharedArgs {
  XpDecodeAttnArgs a;         /* ws: partial sums [batch, q_heads, max_parts + own_slots, head_dim], then their (maximum, sum) pairs
                                 [batch, q_heads, max_parts + own_slots, 2], then batch + 4 words. num_splits and chunk_tokens
                                 (and ws as they want it) are read where max_pieces is 0 */
  const XpPrefixPiece* pieces;
  const int* n_pieces;        /* device words: number of pieces, tokens of the longest one */
  const int* row_prefix;      /* [plan_rows] tokens that a row shares (a multiple of 16); a row of fewer tokens reads all on its own */
  const int* row_parts;       /* [plan_rows] pieces of the row */
  int max_pieces;             /* bound of *n_pieces */
  int max_parts;              /* bound of row_parts, up to XP_PREFIX_PARTS */
  int plan_rows;              /* rows behind these share nothing */
  int own_slots;              /* partial results of a row's own tokens, 2 to XP_PREFIX_OWN */
  int max_len;                /* bound of the sequences' lengths: rows are read no further */
  int reserved;
} XpDecodeSharedArgs;
#define XP_PREFIX_PARTS 32
#define XP_PREFIX_OWN 64
#define XP_PREFIX_ROWS 4096   /* largest batch */
int xp_decode_shared(const XpDecodeSharedArgs* a, void* stream);

/* out[r] = y[r] + scale[s] B[s] (A[s] x[r]) with s the adapter slot of row r (none: out[r] = y[r]). A projection may have several
 * parts, each with its own A and its own features: A's rows and the ranks lie part after part. */
#define XP_LORA_PARTS 4
typedef struct XpLoraItem {
  int slot;                   /* adapter, or -1: rows without one */
  int first, rows;            /* rows perm[first .. first + rows) */
  int pad;
} XpLoraItem;

typedef struct XpLoraArgs {
  const void* x;              /* bf16 [rows, ldx] */
  const void* y;              /* bf16 [rows, ld_y] */
  void* out;                  /* bf16 [rows, ld_out]; may be y */
  int rows, ldx, ld_y, ld_out;
  const XpLoraItem* items;
  const int* n_items;         /* device word */
  const int* perm;            /* [rows] */
  int max_items, reserved;
  /* bf16 [slots, parts, k / 32 rounded up, rank / 8, 8 ranks, 32 of k (zeros behind the last)] */
  const void* a;
  /* bf16, n * rank elements per slot, of which n * ranks[slot] are used, without gaps: blocks of up to 32 features of a part, in
     each [ranks / 16][2][e: feature / 8][2][4 of 4 ranks][2][4 ranks], the twos being bit 2, bit 0 and bit 1 of the feature */
  const void* b;
  const float* scale;         /* [slots] */
  const int* ranks;           /* [slots] rank in use, rounded up to 16; what lies behind it is zero */
  const int* part_ranks;      /* [slots, XP_LORA_PARTS] the parts' own ranks (0: none) */
  int k, n, rank, parts, slots;
  int part_end[XP_LORA_PARTS]; /* features [0, part_end[0]) are part 0, and so on; multiples of 8 */
} XpLoraArgs;
int xp_lora(const XpLoraArgs* a, void* stream);

/* Controls on logits; every array may be null. Order: repetition, frequency, presence, bias, mask. */
typedef struct XpLogitControls {
  const int* history;         /* [history_slots, ld_history] tokens; ids outside the vocabulary count for nothing */
  const int* history_rows;    /* [rows] slot of a row (null: row r is slot r) */
  const int* lens;            /* [rows] tokens in the history */
  const int* prompt_lens;     /* [rows] how many of them are the prompt's (null: none) */
  const int* latest;          /* [rows] the last of the `lens` tokens, not stored yet: the call stores it (null: all are stored) */
  const float* repetition;    /* [rows] a token that occurred: logit > 0 divided by it, others multiplied */
  const float* frequency;     /* [rows] subtracted once for every occurrence behind the prompt */
  const float* presence;      /* [rows] subtracted once if there is any */
  const int* bias_ids;        /* [bias_total] rows one after the other: entries [bias_starts[r], bias_starts[r + 1]) */
  const float* bias_values;
  const int* bias_starts;     /* [rows + 1] */
  const uint32_t* masks;      /* [mask_count, ld_mask] bit i % 32 of word i / 32: token i is allowed */
  const int* mask_index;      /* [rows] mask of a row, outside [0, mask_count): none */
  int history_slots, history_cap, ld_history, bias_total, mask_count, ld_mask;
} XpLogitControls;

typedef struct XpLogitArgs {
  XpLogitControls c;
  const void* logits;         /* [rows, ld] bf16 or fp32 */
  void* out;                  /* adjusted logits [rows, ld_out], bf16 or fp32; null: tokens are selected instead */
  const float* temps;         /* [rows] temperature (null or <= 0: the largest logit, ties to the lower id) */
  const uint32_t* seeds;      /* [rows, 2] */
  int* tokens;                /* [rows] */
  float* values;              /* [rows] optional: the adjusted logit of the selected token */
  int rows, vocab, ld, ld_out, f32, out_f32;
} XpLogitArgs;
#define XP_LOGIT_VOCAB (1 << 20)
int xp_logit_controls(const XpLogitArgs* a, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* XPOOL_REQUEST_API_H_ */
