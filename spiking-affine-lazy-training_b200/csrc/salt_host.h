// The calling thread's error text and launch count, kept in salt_capi.cu, for the other host files.
#pragma once
#include <string>

#include "../../include/salt_b200.h"

namespace salt {

salt_status host_fail(salt_status s, const std::string& msg);  // salt_last_error(); returns s
void host_launched(int n);                                     // salt_launch_counter()

}  // namespace salt
