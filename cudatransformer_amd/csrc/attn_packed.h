// Attention on packed sequences: the plan's layout and the launcher interface between the C-ABI
// layer (packed_capi.hip) and the kernels (attn_packed.hip, attn_packed_generic.hip).
//
// Sequences of different lengths lie one behind the other in [tokens, heads, d] tensors; every
// one attends to itself alone.  Hq query heads share Hkv key / value heads, G = Hq / Hkv
// ("group") to one.  The kernels treat the G query heads of a key head as rows of one matrix:
// row r of a sequence is token r / G, query head kvh * G + r % G, so that a tile of rows reads
// each key block once for the whole group and short sequences fill tiles G times better.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ctattn {

// ---- the plan: one buffer, a host copy that launchers read and a device copy that kernels read.
// PackedHeader, then int32 cu[nseq + 1] (first token of each sequence), then the tables of work
// items.  A table lists the tiles of all sequences for one tile height, the longest running
// first, so that the last workgroups to start are short ones.
struct PackedItem {
    int32_t start;  // first token of the sequence
    int32_t len;    // its tokens
    int32_t tile;   // the tile within it
    int32_t seq;
};
// Tile kinds: rows of (token, head of the group) for the forward and dQ, keys for dK / dV.
enum PackedTile { kRows32 = 0, kRows64, kRows128, kKeys32, kKeys64, kKeys128, kPackedTiles };
constexpr int kPackedTileSize[kPackedTiles] = {32, 64, 128, 32, 64, 128};

struct PackedTable {
    int64_t offset;  // bytes from the start of the buffer
    int64_t count;
};
struct PackedHeader {
    int64_t magic;
    int64_t bytes;
    int64_t nseq, tokens, max_len, group;
    int64_t cu_offset;
    int64_t pairs, pairs_causal;  // (query token, key) pairs within sequences, unmasked and causal
    PackedTable table[2][kPackedTiles];  // [causal][kind]
};
constexpr int64_t kPackedMagic = 0x63746b6470616b31ll;

// Element strides of a [tokens, heads, d] tensor whose last dimension is contiguous.
struct PackedStride {
    int64_t row, head;
};

struct PackedCall {
    int dtype;  // 0 fp32, 1 bf16, 2 fp16, 3 fp64
    const PackedHeader *host;
    const char *dev;
    int64_t hq, hkv, d;
    bool causal;
    PackedStride sq, sk, sv, so, sdo, sdq, sdk, sdv;
    int64_t tokens() const { return host->tokens; }
    int64_t group() const { return host->group; }
    const PackedItem *items(PackedTile kind) const {
        return reinterpret_cast<const PackedItem *>(dev + host->table[causal ? 1 : 0][kind].offset);
    }
    int64_t item_count(PackedTile kind) const { return host->table[causal ? 1 : 0][kind].count; }
};

// ---- generic kernels: any 1 <= d <= 256, any type, any alignment and strides.  lse is
// [tokens, hq], delta scratch of the same shape; both fp64 for dtype 3 and fp32 otherwise. ----
hipError_t launch_packed_generic_fwd(const PackedCall &c, const void *q, const void *k, const void *v, void *o,
                                     void *lse, hipStream_t stream);
hipError_t launch_packed_generic_bwd(const PackedCall &c, const void *q, const void *k, const void *v, const void *o,
                                     const void *dout, const void *lse, void *delta, void *dq, void *dk, void *dv,
                                     hipStream_t stream);

// ---- MFMA kernels: fp32, bf16, fp16; d whole 16-byte chunks up to 128; base pointers and row and head
// strides of q, k, v, o, dout on 16 bytes, of dq, dk, dv on 16 bytes too.  lse may be NULL in the forward. ----
constexpr int64_t kMfmaMaxGroup = 128;
bool packed_mfma_supported(int dtype, int64_t d, int64_t group);
int64_t packed_bwd_scratch_bytes(const PackedCall &c);
hipError_t launch_packed_fwd(const PackedCall &c, const void *q, const void *k, const void *v, void *o, float *lse,
                             hipStream_t stream);
hipError_t launch_packed_bwd(const PackedCall &c, const void *q, const void *k, const void *v, const void *o,
                             const void *dout, const float *lse, void *scratch, void *dq, void *dk, void *dv,
                             hipStream_t stream);

}  // namespace ctattn
