// Byte layout of a granule (16 tokens of one key/value head) of the paged 4-bit cache, shared by the
// launches that write and read it; paged.cu describes it.
#pragma once

#include <stdint.h>

namespace df {
namespace paged {

constexpr int HEAD_DIM = 128;
constexpr int GRANULE = 16;                                // tokens
constexpr int CODE_BYTES = HEAD_DIM / 2;                   // of one token's key or value
constexpr int PARAM_OFFSET = GRANULE * CODE_BYTES;         // (scale, minimum) pairs behind the codes
constexpr int HALF_GRANULE = PARAM_OFFSET + GRANULE * 4;   // keys; the values follow
constexpr int GRANULE_BYTES = 2 * HALF_GRANULE;            // 2176
constexpr int TOKEN_BYTES = GRANULE_BYTES / GRANULE;       // 136

// Where 16-byte chunk c of token r of a granule is stored.
__host__ __device__ constexpr int chunk_place(int c, int r) { return c ^ ((r >> 1) & 3); }

}  // namespace paged
}  // namespace df
