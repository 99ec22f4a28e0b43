// paged.cuh -- declarations shared by the serving-step kernels (rotation, append, attention over a
// shared prefix and paged tails) and their host code.
#pragma once

#include "common.cuh"

namespace kvx {

// Page lookup: token -> (page of the table, place in it).
struct PageSplit {
    int32_t tokens;  // per page
    int32_t shift;   // log2(tokens) when it is a power of two, else -1
    __device__ __forceinline__ void at(int64_t t, int64_t &page, int32_t &place) const {
        if (shift >= 0) {
            page = t >> shift;
            place = int32_t(t & (tokens - 1));
        } else if (t < int64_t(1) << 31) {  // a 32-bit division is several times cheaper
            const uint32_t p = uint32_t(t) / uint32_t(tokens);
            page = p;
            place = int32_t(uint32_t(t) - p * uint32_t(tokens));
        } else {
            page = t / tokens;
            place = int32_t(t - page * tokens);
        }
    }
};

struct PoolDev {
    uint16_t *k, *v;
    int64_t page_stride, token_stride, head_stride;  // elements
    int32_t n_pages;
    PageSplit split;
};

// One kind of head of a rotate / append launch.
struct RotSeg {
    const uint16_t *src;
    uint16_t *dst;          // null: into the pools
    int64_t src_token, src_head, dst_token, dst_head;
    int32_t heads;
    int32_t rotated;        // 0: copied as it is
    int32_t pool;           // 0: dst; 1: K pool; 2: V pool
};

struct RotArgs {
    RotSeg seg[3];
    const float *cos, *sin;
    const int32_t *pos;
    const uint8_t *axis;
    int64_t pos_stride;
    const int64_t *slots;
    PoolDev pool;
    int *status;
    int32_t n_pos, rot_dim, n_axes, interleaved, inverse;
    int32_t n_tokens, dim, heads;    // heads: of all segments together
    int32_t tokens_per_cta, head_slots;
};

cudaError_t launch_rotate(int dtype, bool vec, const RotArgs &a, cudaStream_t s);

// 16 tokens of one tensor of an XKV prefix, as the loader warps of the prefix kernel take them
// (built once by kvx_prefix_create; 32 bytes for 16 tokens).
struct XkvGroup {
    uint64_t rows;    // first token's sign/mantissa bytes, down to the 16-byte line they start in (raw block:
                      // address of its BF16 values)
    uint64_t codes;   // its residual codes, likewise
    uint32_t esc;     // first escape entry (index in XkvDev::esc)
    uint32_t b7;      // the block's merge words (index in XkvDev::b7)
    uint16_t n_rows;  // bytes to copy from rows and from codes (multiples of 16; 0: nothing, a raw block or
    uint16_t n_codes; // no tokens)
    uint32_t bits;    // escapes | tokens << 13 | mode << 18 | offset of the rows << 20 | of the codes << 23 (both even)
    __host__ __device__ int n_esc() const { return int(bits & 0x1FFFu); }
    __host__ __device__ int n() const { return int((bits >> 13) & 31u); }     // 0 past the block's end
    __host__ __device__ int mode() const { return int((bits >> 18) & 7u); }   // 0 raw, 2, 3, 4
    __host__ __device__ uint32_t row_off() const { return (bits >> 20) & 14u; }
    __host__ __device__ uint32_t code_off() const { return (bits >> 23) & 14u; }
};
static_assert(sizeof(XkvGroup) == 32, "XkvGroup is 32 bytes");

// An XKV prefix: every block takes the same number of tiles of kPrefixTile tokens (fewer tokens or none
// in the last ones), every tile a group for each 16 tokens and tensor.
struct XkvDev {
    const XkvGroup *groups;      // [kv head][tile][K, V][kPrefixTile / 16]
    const uint8_t *tile_tokens;  // [kv head][tile]
    const uint32_t *esc, *b7;
    int32_t head_tiles;          // of a head (0: no XKV prefix)
    int32_t tiles;               // up to the last with tokens
};

// One attention call (kvx_batch_attend) as its kernels see it.
struct PagedArgs {
    const uint16_t *q;
    uint16_t *out;
    float *lse;
    int64_t q_token, q_head, out_token, out_head;
    PoolDev pool;
    const int32_t *prefix_table, *table, *lens;
    int64_t table_stride;
    int32_t prefix_len, max_len;
    XkvDev xkv;             // the prefix when xkv.tiles > 0
    int32_t batch, n_q_heads, n_kv_heads, group;
    float scale_log2;       // scale * log2(e)
    int32_t wait_us;        // limit of a wait in the tensor-core prefix kernel (0: nothing is computed)
    int *status;
    // Partial states: row r has dim accumulators at acc + r * dim and {m (log2 units), l} at ml[r].
    float *acc;
    float2 *ml;
    // Tensor-core prefix parts: row ((kv head * n_split + split) * row_pad + row), n_split parts of
    // split_tiles tiles of kPrefixTile tokens (the last fewer) of prefix_tiles for each of the head's
    // batch * group rows, in row_groups items of kPrefixRows rows.
    int32_t n_split, row_pad, split_tiles, prefix_tiles, row_groups;
    int32_t box_tokens, heads_inside;   // TMA boxes of the pools (see the kernel)
    // Streamed units, laid end to end in 16-token tiles: first (a streamed prefix) KV head by KV
    // head and group of 8 rows, prefix_len tokens each; then sequence by sequence, KV head by KV
    // head, group of 8 heads by group, the sequence's own tokens; each unit's tiles are followed by
    // kUnitTiles empty positions.  The line is cut into equal runs; the part that run r
    // leaves of unit u is in rows stream_base + 8 (r + u) .., which no other pair has (r + u grows along
    // the line).
    int64_t stream_base;
    int32_t stream_prefix;  // units of a streamed prefix (0: the prefix is not streamed)
    int32_t pre_groups;     // its groups of 8 rows
    int32_t tail_groups;    // groups of 8 heads of a KV head
    int32_t stream_ctas;    // of kStreamWarps warps
    int32_t stream_runs;
    int32_t shared_runs;    // 0: warp i of the grid takes run i; 1: the warps take runs from next_run
    int32_t *next_run;      // 0 before the call, and again after it
    int32_t *starts;        // [batch + 1] positions of a unit of each sequence before, for the combine
};

constexpr int kStreamWarps = 4;   // a CTA
constexpr int kStreamTile = 16;   // tokens
// Positions a unit takes besides its tiles: its queries' loads, the walk to it and the write of its
// state take a warp about as long as three tiles.  (Without them a warp whose run met a dozen short
// sequences ended 40 us after the others.)
constexpr int kUnitTiles = 3;
constexpr int kMaxStreamBatch = 2048;

// Query rows of an item and tokens of a tile of the tensor-core prefix kernel.
constexpr int kPrefixRows = 128, kPrefixTile = 64;
int prefix_ctas_per_sm(int dim, bool coded);

// What the kernels of a head dim and type need once on a device before they are launched there (shared
// memory beyond the default, which belongs to the device).
cudaError_t prepare_paged_prefix(int dim, int dtype);
cudaError_t prepare_paged_stream(int dim, int dtype);
// The tensor-core kernel over the prefix items of `a`.
cudaError_t launch_paged_prefix(int dim, int dtype, const PagedArgs &a, cudaStream_t s);
// The group table of an XKV prefix from its flat blocks' descriptors (heads * blocks of them).
struct BlockDesc;
cudaError_t launch_xkv_groups(const BlockDesc *desc, int64_t n_blocks, int tiles_per_block, int dim, XkvGroup *groups,
                              uint8_t *tile_tokens, cudaStream_t s);
// The streaming kernel over the units of `a` and the combine pass over every (sequence, head).
// beside: the launch before it on the stream is the same call's prefix kernel, which it may run beside.
cudaError_t launch_paged_stream(int dim, int dtype, const PagedArgs &a, bool beside, cudaStream_t s);
cudaError_t launch_paged_combine(int dim, int dtype, const PagedArgs &a, cudaStream_t s);

}  // namespace kvx
