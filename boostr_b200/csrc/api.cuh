// What the translation units of the C ABI share with api.cu.  Host side only.
#pragma once

namespace b200q {

int api_fail(int code, const char* fmt, ...);  // sets the thread's error text and returns `code`
unsigned int* api_status();                    // device address of the status word of the current device (nullptr: no device)
int api_sm_count();                            // SMs of the current device

}  // namespace b200q
