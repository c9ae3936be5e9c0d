// The paged cache of keys and values held in 4 bits: where everything lies in a page (host and device).
#ifndef ITEXHIP_KV4_HPP_
#define ITEXHIP_KV4_HPP_

#include <stdint.h>

#include "itexhip.h"

namespace itexhip {

#ifdef __HIPCC__
#define KV4_FN __host__ __device__ __forceinline__
#else
#define KV4_FN inline
#endif

// A head padded to what the attention kernels are built for
KV4_FN constexpr int kv4_padded(int head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }

// A page's block of one kv head: key codes, value codes, key parameters, value parameters.  Offsets in bytes from the block.
struct Kv4Block {
  int page_size, dp;
  KV4_FN int bytes() const { return page_size * (dp + 8); }
  KV4_FN int key_codes(int token) const { return token * (dp / 2); }
  // the dword of a token that holds dimensions 8 dword .. 8 dword + 7
  KV4_FN int value_codes(int token, int dword) const {
    return page_size * (dp / 2) + (((token >> 2) * (dp / 8) + dword) * 4 + (token & 3)) * 4;
  }
  KV4_FN int key_params(int token) const { return page_size * dp + (token >> 2) * 16 + (token & 3) * 2; }  // offset: + 8
  KV4_FN int value_params(int token) const { return page_size * (dp + 4) + (token >> 2) * 16 + (token & 3) * 2; }
};

inline int log2_of(int power_of_two) { return __builtin_ctz(static_cast<unsigned>(power_of_two)); }

// nullptr if the geometry is a cache's, else what is wrong with it
inline const char* kv4_invalid(const itexhip_kv4_cache* c) {
  if (c == nullptr) return "null geometry";
  if (c->head_dim < 8 || c->head_dim > 256 || c->head_dim % 8 != 0) return "head_dim is a multiple of 8 from 8 to 256";
  if (c->kv_heads < 1 || c->kv_heads > 65535) return "kv_heads is 1 to 65535";
  if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)) != 0) return "page_size is 16, 32, 64, 128 or 256";
  if (c->num_pages < 1 || c->num_pages > (1ll << 31) - 1) return "num_pages is 1 to 2^31 - 1";
  return nullptr;
}

}  // namespace itexhip
#endif  // ITEXHIP_KV4_HPP_
