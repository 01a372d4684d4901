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


# Calls that need scratch for each of its uses, on addresses that are no memory: the gradient ahead of an activation, columns' sums, both projections' gradients,
# sums of a product whose k is split, rows that begin at odd elements.
CALLS = """
p = 1 << 20
calls = [
    lambda m=4096: w.tiramisu_hip_linear_backward(p, p, p, p, p, p, p, m, 1024, 512, 0, 0, 0, 0, 2, 2),
    lambda m=4096: w.tiramisu_hip_linear_backward(p, p, p, None, p, p, p, m, 1024, 512, 0, 0, 0, 0, 0, 2),
    lambda m=4096: w.tiramisu_hip_gated_linear_backward(p, p, p, p, p, p, p, p, p, m, 1024, 512, 0, 0, 0, 0, 0, 0, 4, 2),
    lambda m=4096: w.tiramisu_hip_rms_norm_backward(p, p, p, p, None, p, p, m, 1024, 0, 0, 0, 2),
    lambda m=4096: w.tiramisu_hip_rms_norm_backward(p, p, p, p, None, p, p, m, 40000, 0, 0, 0, 2),
    lambda m=100: w.tiramisu_hip_linear(p, p, None, None, None, None, p, None, m, 512, 8192, 0, 0, 0, 0, 2, 2),
    lambda m=4096: w.tiramisu_hip_linear(p, p, None, None, None, None, p, None, m, 1024, 513, 0, 0, 0, 0, 2, 2),
    lambda m=4096: w.tiramisu_hip_gated_linear(p, p, p, None, None, None, p, None, None, m, 1024, 513, 0, 0, 0, 4, 2, 2),
]
"""


def test_a_call_without_memory_is_refused():
    """1 and a message, nothing launched, and the process goes on; with memory the same calls run."""
    out, r = host_runtime.run(CALLS + """
hip.recording_memory(1 << 10)
for call in calls:
    print(call(), launches(), hip.recording_held())
hip.recording_memory(1 << 40)
print([call() for call in calls], len(launches()) >= len(calls))
""")
    assert r.returncode == 0, r.stderr
    assert out == "1 [] 0\n" * 8 + "[0, 0, 0, 0, 0, 0, 0, 0] True\n"
    assert r.stderr.count(" bytes of scratch") == 8


def test_idle_blocks_make_room():
    assert host_runtime.printed(CALLS + """
hip.recording_memory(100 << 20)
w.tiramisu_hip_free(w.tiramisu_hip_malloc(95 << 20))
print(hip.recording_held() >> 20, calls[2](), hip.recording_held() <= 20 << 20)
""") == "95 0 True\n"


def test_scratch_of_varying_sizes_is_little_more_than_the_largest():
    assert host_runtime.printed(CALLS + """
for m in list(range(64, 20000, 333)) + list(range(20000, 64, -333)):
    for call in calls[:4]:
        assert call(m) == 0
held, before = hip.recording_held(), hip.recording_allocations()
for m in range(64, 20000, 777):
    for call in calls[:4]:
        assert call(m) == 0
print(hip.recording_allocations() == before, w.tiramisu_hip_cached_memory_bytes() == held, w.tiramisu_hip_release_cached_memory() == held, hip.recording_held())
calls[2](20000)
print(20000 * 4096 <= hip.recording_held(), held <= 1.13 * hip.recording_held())
""") == "True True True 0\nTrue True\n"


def test_scratch_of_a_recorded_call_stays():
    """A block that was given while a graph was recorded is not freed when a larger one is needed; one that was not, is."""
    assert host_runtime.printed(CALLS + """
calls[2](64)
small = hip.recording_held()
hip.recording_capture(1)
calls[2](128)
recorded = hip.recording_held()
hip.recording_capture(0)
calls[2](1024)
held = hip.recording_held()
calls[2](4096)
print(recorded > small, held >= recorded + 1024 * 4096, recorded + 4096 * 4096 <= hip.recording_held() < held + 4096 * 4096 * 1.2)
""") == "True True True\n"
