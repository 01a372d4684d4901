"""Where the operators' scratch and the memory that the runtime keeps between calls come from (include/tiramisu_hip_wrappers.h)."""
import host_runtime


def test_kept_memory_belongs_to_a_gpu():
    """One thread, one stream handle (that of every GPU's null stream), two GPUs: a block each, and the same one at the next call."""
    assert host_runtime.printed("""
site = ctypes.c_char()
at = lambda: w.tiramisu_hip_kept_scratch(ctypes.addressof(site), 1 << 20, None)
w.tiramisu_hip_set_stream(w.tiramisu_hip_null_stream())
first = at()
hip.hipSetDevice(1)
second = at()
again = at()
hip.hipSetDevice(0)
print(first != second, again == second, at() == first)
""") == "True True True\n"
