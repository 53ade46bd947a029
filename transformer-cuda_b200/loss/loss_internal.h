// Shared by the translation units of libb200loss; not installed.
#pragma once

namespace b200loss {

// Stores the text that b200loss_last_error() returns on the calling thread: "what", or "what: detail". Never throws.
void set_error(const char* what, const char* detail = nullptr);

}  // namespace b200loss
