// skv_exchange.cuh -- how the two threads of a row exchange a value per tile.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define SKV_ANY_SIDE __host__ __device__
#else
#define SKV_ANY_SIDE
#endif

namespace skv {

// Thread `half` of a row writes its value of tile g to this slot, both meet at
// one barrier, and each reads the other's slot.  The slots change places with
// every tile, so that a thread writes where it read itself a tile before:
// nobody else reads that slot any more, however far the two drift apart
// between barriers.  With slots that stay, a thread that is a barrier ahead
// could overwrite a value before its partner has read it.
SKV_ANY_SIDE constexpr int exchange_slot(int half, uint32_t g) { return half ^ (int)(g & 1); }

}  // namespace skv
