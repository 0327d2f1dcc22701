// The head of a context's workspace, which quant_linear_reset_workspace zeroes and whose status word every kernel with bounded waits
// sets when one of them gives up. What lies behind it is free for one launch sequence at a time on the context's stream.
#pragma once
#include <cstddef>

namespace tts {
namespace b200 {
constexpr size_t kStatusOffset = 16384;    // int status[4]: nonzero after a bounded wait gave up
constexpr size_t kSettleOffset = 16640;    // int: written by quant_linear_settle, read by nobody
constexpr size_t kPassOffset = 16768;      // int: 1 from an attention's first pass until its combine, where a second pass is launched between them
constexpr size_t kWorkspaceHeader = 32768;
} // namespace b200
constexpr size_t quant_linear_header_bytes() { return b200::kWorkspaceHeader; }
inline int *quant_linear_status_word(void *workspace) { return reinterpret_cast<int *>(static_cast<char *>(workspace) + b200::kStatusOffset); }
inline int *attention_pass_word(void *workspace) { return reinterpret_cast<int *>(static_cast<char *>(workspace) + b200::kPassOffset); }
} // namespace tts
