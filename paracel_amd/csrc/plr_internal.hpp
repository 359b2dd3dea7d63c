// What the library's translation units share besides the public header.
#pragma once

// Record `msg` as the description plr_last_error(NULL) gives for a call that takes no context
// and return `code`.  Throws nothing.
__attribute__((visibility("hidden"))) int plr_fail_without_context(int code, const char* msg);
