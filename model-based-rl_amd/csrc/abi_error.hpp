// The text behind mbrl_last_error(), shared by the translation units of libmbrl_hip.so (defined in mbrl_hip.hip).
#pragma once
namespace mbrl {
// Records `text` for the calling thread and returns `code`, so that an entry point can `return report(-7, "...")`.
__attribute__((visibility("hidden"))) int report(int code, const char *text);
}  // namespace mbrl
