// How the other sources of the language-model library report an error: the message that smol_lm_last_error returns (one per thread), and the code.
#pragma once

namespace smol {
namespace lm {
int report(int code, const char* who, const char* what) noexcept;
}
}  // namespace smol
