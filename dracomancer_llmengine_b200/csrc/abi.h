// What the files of C entry points share: the thread's error text, the launch counter, pointer checks (defined in abi.cu).
#pragma once

namespace draco {
void abi_error(const char* text);           // text of draco_b200_last_error()
void abi_count(int kernels);                // adds to draco_b200_launch_count(); waits for no lock
bool abi_device_ptr(const void* p);         // device or managed memory
}  // namespace draco
