// The 4-bit paged KV cache: argument checks and address arithmetic shared by
// its kernels (write/read, attention, page operations).
//
// A (page, head) holds page_size / 16 tiles of 16 tokens.  A tile is
//   keys    16 x 64 bytes, 4 bits a dim
//   values  16 x 64 bytes
//   pairs   16 x [groups key pairs | groups value pairs], fp16 (low, delta)
// with groups = 128 / dim_group_size, so a run of tokens inside a page is one
// contiguous run of bytes (one bulk copy), and a single token is three aligned
// pieces of 64, 64 and 8 * groups bytes.  Row orders (chosen for the fragments
// of the attention's matrix products, see kv4_attention.cu):
//   key words     natural 4-byte word w (dims 8w..8w+7) sits at slot (w % 4) * 4 + w / 4
//   value bytes   natural byte b (dims 2b, 2b+1) sits at byte (b % 8) * 8 + b / 8
#pragma once

#include "common.cuh"

namespace popkv {

constexpr int kKv4Dim = 128;
constexpr int kKv4TileTokens = 16;
constexpr int kKv4RowBytes = 64;                                  // 128 dims of 4 bits
constexpr int kKv4ValueOffset = kKv4TileTokens * kKv4RowBytes;    // within a tile
constexpr int kKv4PairOffset = 2 * kKv4ValueOffset;

constexpr int kKv4StatusFull = 1;     // status[0]: an extend found too few free pages or table columns; extends and
                                      // writes do nothing while it is set
constexpr int kKv4StatusWait = 4;     // status[0]: an attention's wait for its copies gave up
constexpr int kKv4StatusSequence = 2; // status[0]: a sequence or page id was out of range or repeated

struct Kv4View {
    uint8_t* pages;
    int32_t* refs;
    int32_t* lengths;
    int32_t* table;
    int32_t* status;
    int layers, num_pages, kv_heads, page_shift, groups, max_seqs, max_pages;
    int64_t head_bytes;   // one (page, head)
    int64_t page_bytes;   // one page of a layer: kv_heads * head_bytes
    int64_t layer_bytes;  // num_pages * page_bytes

    __host__ __device__ int page_size() const { return 1 << page_shift; }
    __host__ __device__ int pair_bytes() const { return 8 * groups; }
    __host__ __device__ int tile_bytes() const { return kKv4PairOffset + kKv4TileTokens * pair_bytes(); }
    __device__ int pages_of(int tokens) const { return (tokens + page_size() - 1) >> page_shift; }
    __device__ bool has_sequence(int s) const { return s >= 0 && s < max_seqs; }
    // Tokens of sequence s; an id out of range (a padding slot) has none.
    __device__ int length_of(int s) const {
        if (!has_sequence(s)) return 0;
        const int most = max_pages << page_shift;
        const int held = lengths[s];
        return held < 0 ? 0 : held > most ? most : held;
    }
    // Page of a token position of sequence s (both in range), or -1.
    __device__ int page_at(int s, int position) const {
        const int page = table[static_cast<int64_t>(s) * max_pages + (position >> page_shift)];
        return page < num_pages ? page : -1;
    }
    // First byte of the tile that holds `position` in page `page`.
    __device__ uint8_t* tile_at(int layer, int page, int head, int position) const {
        return pages + layer * layer_bytes + page * page_bytes + head * head_bytes +
               ((position & (page_size() - 1)) >> 4) * static_cast<int64_t>(tile_bytes());
    }
};

// Checks the descriptor and fills the view; POPKV_OK or an error status.
int kv4_view(const char* what, const popkv_kv4_cache* cache, Kv4View* view);

// Copies pages from sources[i] to targets[i] (device, skipped where the source is
// negative) in every layer.  `count` is the number of entries; when `count_dev` is
// non-NULL only the first *count_dev of them are copied.
int kv4_copy_launch(const char* what, const Kv4View& view, const int32_t* sources, const int32_t* targets,
                    int64_t count, const int32_t* count_dev, cudaStream_t stream);

}  // namespace popkv
