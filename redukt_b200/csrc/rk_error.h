// The library's error message (redukt_b200_last_error), shared by its translation units.
#pragma once

namespace rk {
void set_err(const char* fmt, ...);
}
