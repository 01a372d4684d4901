"""Where the operators' scratch and the memory that the runtime keeps between calls come from (include/tiramisu_hip_wrappers.h)."""
import pytest
import torch

import host_runtime
from tiramisu_amd import operators, runtime


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


def test_idle_blocks_of_the_pool_belong_to_a_gpu():
    """A block that was freed on one GPU is handed out there only."""
    assert host_runtime.printed("""
first = w.tiramisu_hip_malloc(1 << 20)
w.tiramisu_hip_free(first)
hip.hipSetDevice(1)
second = w.tiramisu_hip_malloc(1 << 20)
hip.hipSetDevice(0)
print(second != first, w.tiramisu_hip_malloc(1 << 20) == first)
w.tiramisu_hip_free(second)
print(w.tiramisu_hip_malloc(1 << 20) != second, w.tiramisu_hip_cached_memory_bytes() == 1 << 20)
hip.hipSetDevice(1)
print(w.tiramisu_hip_malloc(1 << 20) == second, w.tiramisu_hip_release_cached_memory())
""") == "True True\nTrue True\nTrue 0\n"


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


def test_scratch_from_a_source_of_the_callers():
    """Asked once a call, with as much as the call needs; the runtime keeps nothing then, and a source that has nothing refuses the call."""
    assert host_runtime.printed(CALLS + """
class Source(ctypes.Structure):
    _fields_ = [("take", ctypes.CFUNCTYPE(ctypes.c_void_p, ctypes.c_uint64, ctypes.c_void_p)), ("context", ctypes.c_void_p)]
asked = []
def give(bytes, context):
    asked.append(bytes)
    return context
ours = Source(Source._fields_[0][1](give), 1 << 40)
held = Source(ours.take, ours.context)
w.tiramisu_hip_exchange_scratch_source(ctypes.byref(held))
print(bool(held.take), [call() for call in calls], len(asked), min(asked) > 0, hip.recording_held())
print(asked[0] >= 4096 * 1024 * 2, asked[2] >= 4096 * 2048 * 2, asked[6] >= 5120 * 514 * 2)
none = Source(ours.take, None)
w.tiramisu_hip_exchange_scratch_source(ctypes.byref(none))
launches()
print([call() for call in calls], launches())
w.tiramisu_hip_exchange_scratch_source(ctypes.byref(held))
print([call() for call in calls], len(asked), hip.recording_held() > 0)
""") == """False [0, 0, 0, 0, 0, 0, 0, 0] 8 True 0
True True True
[1, 1, 1, 1, 1, 1, 1, 1] []
[0, 0, 0, 0, 0, 0, 0, 0] 16 True
"""


def scratch_inputs(M, N, K, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return [torch.randn(shape, device="cuda", generator=g).bfloat16() for shape in ((M, N), (M, K), (N, K), (M, N))]


@pytest.mark.gpu
def test_scratch_of_tensors_is_torchs():
    """The runtime keeps nothing of calls on tensors, and a later tensor may have the memory."""
    w = runtime.wrappers()
    w.tiramisu_hip_release_cached_memory()
    dy, x, weight, pre = scratch_inputs(301, 1000, 77, 1)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = operators.linear_backward(dy, x, weight, pre=pre, activation="gelu", bias=True)
    assert w.tiramisu_hip_cached_memory_bytes() == 0
    results = sum((t.numel() * 2 + 511) // 512 * 512 for t in got)
    assert torch.cuda.memory_allocated() == before + results and torch.cuda.max_memory_allocated() >= before + results + 301 * 1000 * 2


@pytest.mark.gpu
def test_no_memory_is_an_exception():
    """Scratch that torch has no memory for: torch's exception, and the same call runs where there is some."""
    dy, x, weight, pre = [torch.randn(shape, device="cuda", dtype=torch.bfloat16) for shape in ((1 << 16, 4096), (1 << 16, 64), (4096, 64), (1 << 16, 4096))]
    expected = operators.linear_backward(dy, x, weight, pre=pre, activation="silu")
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    held = []
    try:
        # room for the results, 9 MiB, but not for 520 MiB of scratch: what is left within torch's own blocks is taken
        torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (64 << 20)) / torch.cuda.get_device_properties(0).total_memory)
        with pytest.raises(torch.cuda.OutOfMemoryError):
            while True:
                held.append(torch.empty(256 << 20, dtype=torch.uint8, device="cuda"))
        with pytest.raises(torch.cuda.OutOfMemoryError, match="520.00 MiB"):
            operators.linear_backward(dy, x, weight, pre=pre, activation="silu")
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
        held.clear()
    for got, was in zip(operators.linear_backward(dy, x, weight, pre=pre, activation="silu")[:2], expected):
        assert torch.equal(got, was)


@pytest.mark.gpu
def test_graphs_of_one_recording_stream_replay_beside_each_other():
    """Two graphs, recorded one after the other on the stream that torch records on, replayed at the same time on two streams: each has scratch of its own."""
    shapes = [(900, 1003, 512), (700, 1203, 512)]
    inputs = [scratch_inputs(*shape, seed) for seed, shape in enumerate(shapes)]

    def call(dy, x, weight, pre):
        return operators.linear_backward(dy, x, weight, pre=pre, activation="gelu", bias=True)

    expected = [call(*t) for t in inputs]
    graphs, results = [], []
    for t in inputs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            results.append(call(*t))
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for turn in range(3):
        for r in results:
            for t in r:
                t.zero_()
        torch.cuda.synchronize()
        for _ in range(20):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for got, was in zip(results, expected):
            assert all(torch.equal(u, v) for u, v in zip(got, was))
        call(*inputs[turn % 2])


def test_launches_hold_fewer_than_2_to_the_32_threads():
    """Rows of a workgroup of 1024 threads each, just more than one launch holds: several launches, which together are all of the rows'."""
    out = host_runtime.printed("""
p = 1 << 20
rows = (1 << 22) + 5
def rows_of(kernel):
    found = [b for k, b, t in launches() if kernel in k]
    return len(found), sum(found)
for type, columns in ((2, 8200), (0, 4100), (2, 40000)):
    assert w.tiramisu_hip_quantize_rows(p, p, p, rows, columns, 0, type) == 0
    print(rows_of("rms_norm_kernel"))
assert w.tiramisu_hip_rms_norm(p, p, p, p, p, None, p, rows - 5, 8200, 0, 0, 1e-6, 2, 2) == 0
print(rows_of("rms_norm_kernel"))
assert w.tiramisu_hip_rms_norm_backward(p, p, p, p, p, p, p, rows, 40000, 0, 0, 0, 2) == 0
print(rows_of("long_rows"))
""")
    rows = (1 << 22) + 5
    assert out == ("(2, %d)\n" % rows) * 3 + "(2, %d)\n" % (rows - 5) + "(2, %d)\n" % rows


def test_gradients_of_overlapping_rows_are_refused():
    """dx and dweight read their operands down the columns, up to an end behind the last row: rows closer together than they are long have none."""
    out, r = host_runtime.run("""
p = 1 << 20
print([w.tiramisu_hip_linear_backward(p, p, p, None, p, p, None, 70, 40, 50, *strides, 0, 0, 2) for strides in ((39, 0, 0), (0, 49, 0), (0, 0, 1), (40, 50, 50))])
print([w.tiramisu_hip_gated_linear_backward(p, p, p, p, p, p, p, p, p, 70, 40, 50, 0, *strides, 0, 0, 4, 2) for strides in ((49, 0, 0), (0, 49, 0), (0, 0, 49), (50, 51, 52))])
print(w.tiramisu_hip_linear_backward(p, p, p, None, p, p, None, 1, 40, 50, 1, 1, 0, 0, 0, 2))
""")
    assert r.returncode == 0 and out == "[1, 1, 1, 0]\n[1, 1, 1, 0]\n0\n", r.stderr
    assert r.stderr.count(" apart") == 6
