// The operators of a decoder's attention block (include/wkf_decode.h): what their handles hold and what their graph
// nodes carry.
#pragma once

#include <cstdint>
#include <memory>
#include <mutex>
#include <vector>

#include "core.h"

namespace wkf {

// Most sequences of a cache, and most batch entries of one norm_rope launch: their lengths travel in the launch's
// argument block.
constexpr size_t kMaxSequences = 256;

// A matrix W [k, n] in 4 bits, laid out as the B operands of 16x16x32 MFMAs read it.
// codes: tiles of 16 columns x 128 rows, [n/16][k/128], 1 KiB each; lane l of a wave owns 16 bytes of a tile, word w of
//   which holds column l % 16, rows 32 w + 8 (l / 16) + e for e = 0..7: the even e in nibbles 0..3, the odd e in nibbles 4..7
//   (so that one mask leaves two neighbouring elements in the two halves of a register).
// scales, zeros: [n/16][groups][16], the scales in their own type, a zero point a byte.
struct Q4 {
  wkf_device* dev = nullptr;
  size_t k = 0, n = 0, group = 0, groups = 0;  // group: at most k rounded up to 32
  size_t given_group = 0;
  DType scale_dtype = DType::F16;
  BufRef codes, scales, zeros;  // zeros: none = 8 everywhere
  bool fits_f16 = false;        // every weight is zero, or within the normal numbers of f16 when it is rounded to that
  size_t tiles_k() const { return (k + 127) / 128; }
  size_t tiles_n() const { return (n + 15) / 16; }
};

// Keys and values in 8 bits.  codes: [keys | values][sequence][head], each cap x dp bytes in MFMA order (see
// kernels/kv_layout.hip.inc); scales: [keys | values][sequence][head][cap / block]; staged: the originals of the unfinished
// block, [slot][keys | values][sequence][head][block][dim] f32.  A block that is begun by the append that finishes another
// goes to the other slot: the workgroup that finishes the first still reads it.
struct KvCache {
  wkf_device* dev = nullptr;
  size_t seqs = 0, heads = 0, dim = 0, dp = 0, block = 0;
  size_t capacity = 0, cap = 0;  // tokens of a sequence: what was asked for, and rounded up to whole blocks and to 64
  BufRef codes, scales, staged;
  BufRef done;          // split attention: parts finished, a counter for each workgroup
  size_t counters = 0;
  std::mutex mu;  // lengths, slots and generation; held while a launch that goes by them is put on the stream
  std::vector<uint32_t> len;
  std::vector<uint8_t> slot;
  uint64_t generation = 0;  // counts appends and resets: a node recorded before one is refused after it
};

struct Q4Args : DecodeArgs {
  std::shared_ptr<const Q4> w;
};

struct NormRopeArgs : DecodeArgs {
  float eps = 0.f;
  std::vector<uint32_t> positions;  // one a batch entry
};

struct CacheArgs : DecodeArgs {  // CacheValues, Attend
  std::shared_ptr<KvCache> c;
  uint64_t generation = 0;
  size_t first = 0, count = 0;      // CacheValues
  float scale = 0.f;                // Attend
  bool causal = true;
  std::vector<uint32_t> counts;
};

}  // namespace wkf
