/*
 * C ABI of the paged key/value cache operators for B200 (sm_100a): what a decoding server does around
 * the masked attention of fa_mask_fwd_sm100.h.  The reference has no counterpart for any of them.
 *
 *   fa_paged_extend_sm100     block tables, slots and positions of new tokens from request lengths
 *   fa_paged_shrink_sm100     the way back: pages behind a shorter length return to the free list
 *   fa_rotary_sm100           rotary positions on queries and keys in the attention's layout
 *   fa_paged_append_sm100     rotary positions on new tokens, keys and values written into the pages
 *   fa_paged_attention_sm100  attention of one new token per request over the pages
 *
 * Conventions are those of fa_mask_fwd_sm100.h: every function returns FA_PAGED_OK (0) or a negative
 * FA_PAGED_ERR_* code, never throws, never synchronises, never allocates; memory belongs to the caller;
 * work is enqueued on the caller's stream, chained to the kernel before it (every kernel waits for that
 * one before it touches memory).  No kernel here waits for another one's memory, so there is no status
 * word.  The first call of an operator with given types, shapes and options loads its kernel: make it outside any stream
 * capture.  Pointers are device pointers on `device`; `struct_size` is sizeof of the struct, checked.
 *
 * The cache: pages of `page_size` tokens, k and v each (num_pages, heads_k, page_size, head_dim) of one
 * 16-bit type, addressed through their element strides (page, head, token); the last dimension is
 * contiguous, the strides are multiples of 8 elements and the bases 16-byte aligned, so a
 * (num_pages, page_size, heads_k, head_dim) layout or one layer of a larger array serves as well.
 * Slot s of the cache is token s % page_size of page s / page_size.  Row b of the block table names the
 * pages of request b in order.
 */
#ifndef FA_PAGED_SM100_H_
#define FA_PAGED_SM100_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define FA_PAGED_ABI_VERSION 1

enum {
    FA_PAGED_OK = 0,
    FA_PAGED_ERR_NULL = -1,       /* a required pointer is NULL */
    FA_PAGED_ERR_DTYPE = -2,      /* dtype is neither FA_PAGED_FP16 nor FA_PAGED_BF16 */
    FA_PAGED_ERR_SHAPE = -3,      /* a size is negative, too large, or does not divide another */
    FA_PAGED_ERR_HEAD_DIM = -4,   /* head_dim is neither 64 nor 128 */
    FA_PAGED_ERR_ALIGN = -5,      /* a base is not 16-byte aligned or a stride no multiple of 8 elements */
    FA_PAGED_ERR_WORKSPACE = -6,  /* workspace missing, misaligned or too small */
    FA_PAGED_ERR_ARCH = -7,       /* the device is not compute capability 10.x */
    FA_PAGED_ERR_CUDA = -8,       /* a CUDA runtime call failed */
    FA_PAGED_ERR_ROTARY = -9,     /* rot_dim is odd, below 2 or above head_dim */
    FA_PAGED_ERR_SCORE = -10,     /* scale, softcap or window is negative or not finite */
    FA_PAGED_ERR_ABI = -11        /* struct_size does not match this library */
};

enum { FA_PAGED_FP16 = 0, FA_PAGED_BF16 = 1 };

/* Most requests of one extend or shrink call: their prefix sums live in one SM's shared memory. */
#define FA_PAGED_MAX_REQUESTS 16384

typedef struct FaPagedCache {
    void* k;
    void* v;
    int64_t k_page_stride, k_head_stride, k_row_stride;   /* elements */
    int64_t v_page_stride, v_head_stride, v_row_stride;
    int32_t num_pages;
    int32_t heads_k;
    int32_t page_size;
    int32_t head_dim;
} FaPagedCache;

/*
 * Request b holds lens[b] tokens and gets new_lens[b] more (negative lengths count as 0).  It needs
 * ceil((lens + new) / page_size) - ceil(lens / page_size) pages, which are free_pages[head], [head + 1],
 * ... in the order of the requests.  A request is refused as a whole when the table has too few columns
 * for it or the free pages run out - and then so is every later one that needs a page, so what is given
 * does not depend on timing.  Writes
 *   block_table[b]   the new pages behind those the request has; nothing else
 *   lens_out[b]      lens + new, or lens for a refused request
 *   head_out         head + the pages given
 *   cu[0 .. batch]   prefix sums of new_lens: where each request's tokens lie among the packed ones
 *   slots[t]         for t < num_tokens: the token's slot; -1 for a token of a refused request and
 *                    behind the last one (padding)
 *   positions[t]     lens[b] + its index among the request's new tokens; 0 behind the last one
 * The sum of new_lens must be below 2^31.  lens_out may be lens and head_out may be free_head (updated in place).  Requests are extended in full
 * also where num_tokens is smaller than cu[batch].
 */
typedef struct FaPagedExtendArgs {
    uint32_t struct_size;
    int32_t device;
    int32_t* block_table;       /* (batch, table_width), rows table_stride apart */
    int64_t table_stride;
    const int32_t* lens;        /* (batch) */
    const int32_t* new_lens;    /* (batch) */
    const int32_t* free_pages;  /* (num_free_pages) */
    const int32_t* free_head;   /* (1): free_pages before it are taken */
    int32_t* lens_out;          /* (batch) */
    int32_t* head_out;          /* (1) */
    int64_t* slots;             /* (num_tokens) */
    int32_t* positions;         /* (num_tokens) */
    int32_t* cu;                /* (batch + 1) */
    int32_t batch;
    int32_t table_width;
    int32_t page_size;
    int32_t num_free_pages;
    int64_t num_tokens;
} FaPagedExtendArgs;

int fa_paged_extend_sm100(const FaPagedExtendArgs* args, void* stream);

/*
 * Shortens every request to min(lens, keep_lens) tokens (0 releases it) and puts the pages behind that
 * length back in front of free_head, which moves down by their number, so that the next extend takes them
 * again: the free list is a stack.  Updates lens, free_pages and free_head in place; the block table keeps
 * its (now unused) entries.  A head that would become negative - pages that never came from this list - is
 * refused on the device: the pages of the requests that would not fit stay where they are, and the requests
 * keep their length.  A page belongs to one request: one that the caller has put into two rows (a prefix that two
 * requests share) would come back twice, and the next extend would give it to two requests.
 */
typedef struct FaPagedShrinkArgs {
    uint32_t struct_size;
    int32_t device;
    const int32_t* block_table;
    int64_t table_stride;
    int32_t* lens;
    const int32_t* keep_lens;
    int32_t* free_pages;
    int32_t* free_head;
    int32_t batch;
    int32_t table_width;
    int32_t page_size;
    int32_t num_free_pages;
} FaPagedShrinkArgs;

int fa_paged_shrink_sm100(const FaPagedShrinkArgs* args, void* stream);

/*
 * The rotation: elements 0 .. rot_dim - 1 of a head form rot_dim / 2 pairs, (i, i + rot_dim / 2), or
 * (2i, 2i + 1) with `interleaved`; pair i of a token at position p is turned by p * freqs[i] radians and
 * scaled by mscale:  (a, b) -> mscale * (a cos - b sin, b cos + a sin).  `adjoint` turns the other way: the
 * gradient with respect to the input.  Elements from rot_dim on pass through.  Angles are reduced in 64
 * bits, the products are fp32, the result is rounded once.
 */
typedef struct FaRotarySpec {
    const double* freqs;        /* (rot_dim / 2) radians per position */
    const void* positions;      /* int32, or int64 with positions_64 */
    int32_t positions_64;
    int32_t rot_dim;
    int32_t interleaved;
    int32_t adjoint;
    float mscale;
    int32_t reserved;           /* 0 */
} FaRotarySpec;

/*
 * q (batch, heads, seqlen, head_dim), k (batch, heads_k, seqlen, head_dim) through their strides ->
 * q_out, k_out contiguous.  positions[b * position_batch_stride + s].  heads_k may be 0.
 * An output must not overlap an input.  At most FA_ROTARY_MAX_BATCH batch rows a call (a grid's second dimension);
 * the torch operator takes more in several launches.
 */
#define FA_ROTARY_MAX_BATCH 65535
typedef struct FaRotaryArgs {
    uint32_t struct_size;
    int32_t device;
    const void* q;
    const void* k;
    void* q_out;
    void* k_out;
    int64_t q_batch_stride, q_head_stride, q_row_stride;  /* elements, multiples of 8 */
    int64_t k_batch_stride, k_head_stride, k_row_stride;
    int64_t position_batch_stride;
    FaRotarySpec rotary;
    int32_t batch, heads, heads_k, seqlen, head_dim, dtype;
} FaRotaryArgs;

int fa_rotary_sm100(const FaRotaryArgs* args, void* stream);

/*
 * k, v (num_tokens, heads_k, head_dim) through their strides: v goes to cache.v at each token's slot, k -
 * turned, unless rotary.freqs is NULL - to cache.k.  q (num_tokens, heads, head_dim), or NULL with heads = 0, is
 * turned into the contiguous q_out.  A token whose slot is negative or behind the cache is not written (its q
 * is turned all the same).  Two tokens with the same slot: each 16 bytes of the slot are those of one of them.
 */
typedef struct FaPagedAppendArgs {
    uint32_t struct_size;
    int32_t device;
    const void* q;
    const void* k;
    const void* v;
    void* q_out;
    const void* slots;          /* (num_tokens) int64, or int32 with slots_64 = 0 */
    int64_t q_token_stride, q_head_stride;                /* elements, multiples of 8 */
    int64_t k_token_stride, k_head_stride;
    int64_t v_token_stride, v_head_stride;
    FaPagedCache cache;
    FaRotarySpec rotary;
    int64_t num_tokens;
    int32_t heads;
    int32_t dtype;
    int32_t slots_64;
    int32_t reserved;           /* 0 */
} FaPagedAppendArgs;

int fa_paged_append_sm100(const FaPagedAppendArgs* args, void* stream);

/*
 * One new token per request: q (batch, heads, head_dim) attends over the first lens[b] tokens of request b,
 * the last of which is the new one (its key and value are in the cache already); head h reads key head
 * h / (heads / heads_k).  With x = scale * q.k, in this order
 *   softcap > 0:  x = softcap * tanh(x / softcap)
 *   slopes:       x += slopes[h] * (j - (lens[b] - 1))          for key j, a bias by distance
 *   window > 0:   only the last `window` keys are visible
 * out[b, h] = softmax(x) v, lse[b, h] = log(sum(exp(x))) (natural, fp32, optional).  A request without a key
 * gives 0 and -inf.  Lengths are clamped to [0, table_width * page_size]; keys of a page number outside the
 * cache are hidden; what the cache holds behind a request's length or ahead of its window is never used, and
 * only pages with a visible key are looked up.
 * Weights, sums and accumulators are fp32 (a weight enters the product with v as the sum of two 16-bit numbers).
 * The cap adds an error of at most cap * 2^-21 to a score up to a cap of 64, of 2^-18.9 of the score above that.
 * Long histories are split over the GPU and joined through the workspace; the result depends, within the fp32
 * rounding of the join, on how they are split - on the number of SMs, the table's width and the lengths of the other
 * requests of the call - never on timing.  How the work is divided goes by what the table and the window could hold,
 * since the lengths are on the device: a table no wider than the longest request lets short ones be done in one launch.
 * An infinite value that a row sees gives NaN (its weight's second part is 0 or negative).
 */
typedef struct FaPagedAttentionArgs {
    uint32_t struct_size;
    int32_t device;
    const void* q;              /* rows of head_dim, q_batch_stride / q_head_stride elements apart (multiples of 8) */
    void* out;                  /* (batch, heads, head_dim) contiguous, the cache's dtype */
    float* lse;                 /* (batch, heads) or NULL */
    const int32_t* block_table; /* (batch, table_width), rows table_stride apart */
    const int32_t* lens;        /* (batch) */
    const float* slopes;        /* (heads) or NULL */
    int64_t q_batch_stride, q_head_stride;
    int64_t table_stride;
    FaPagedCache cache;
    int32_t batch;
    int32_t heads;
    int32_t table_width;
    int32_t window;
    float scale;
    float softcap;
    int32_t dtype;
    int32_t reserved;           /* 0 */
} FaPagedAttentionArgs;

/* Validates `args` and says how much workspace the call needs (any content, 16-byte aligned, private to the
 * call until it has finished). */
int fa_paged_attention_sm100_workspace_bytes(const FaPagedAttentionArgs* args, size_t* bytes);
int fa_paged_attention_sm100(const FaPagedAttentionArgs* args, void* workspace, size_t workspace_bytes,
                             void* stream);

int fa_paged_sm100_abi_version(void);
/* Kernels this library has launched in this process so far. */
int fa_paged_sm100_launch_count(uint64_t* launches);
const char* fa_paged_sm100_strerror(int code);

#ifdef __cplusplus
}
#endif
#endif /* FA_PAGED_SM100_H_ */
