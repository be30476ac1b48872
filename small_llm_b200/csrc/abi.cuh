// Shared by the translation units behind include/sllm.h.
#pragma once

namespace sllm {

// Keeps the text that sllm_last_error(NULL) returns on this thread; returns `code`.
int fail_text(int code, const char* msg) noexcept;

}  // namespace sllm
