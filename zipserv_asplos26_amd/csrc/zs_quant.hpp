// zs_quant.hpp -- how a quantised paged KV cache is laid out.
//
// The cache is bytes [num_blocks][Hkv][record].  A record holds a page of one KV
// head: first 8 bytes a token, (scale, low) of its key and (scale, low) of its
// value in bf16, then the tokens' rows of key codes and behind them the rows of
// value codes, D bits / 8 bytes each.  A value is low + code scale.
//
// In 4 bits dword j of a row holds channels 8j .. 8j + 7: channel 8j + 2i in bits
// 4i and up, channel 8j + 2i + 1 in bits 16 + 4i and up, so a shift and a mask leave
// two neighbouring channels in the halves of a dword.  In 8 bits channel d is byte d.
//
// So a page of 16 tokens of 128 channels in 4 bits is 17 lines of 128 bytes one
// behind another, and what an attention reads of a token besides its codes comes in
// one piece of 8 bytes.
#pragma once

#include <stdint.h>

namespace zs {

template <int D, int kBits>
struct QuantRow {
  static constexpr int kBytes = D * kBits / 8;  // of a row of codes
};

constexpr int quant_token_bytes(int head_dim, int bits) { return 8 + head_dim * bits / 4; }

}  // namespace zs
