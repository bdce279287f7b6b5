"""Streams and captured graphs of the HIP runtime that the library is linked
with (another copy of the runtime in the process would see no device)."""
import ctypes as C

import nutllm_amd as nut


def _call(name, *args):
    status = getattr(nut.lib(), name)(*args)
    assert status == 0, f"{name}: HIP error {status}"


class Stream:
    """A stream that does not wait for the null stream."""

    def __init__(self):
        self.handle = C.c_void_p()
        _call("hipStreamCreateWithFlags", C.byref(self.handle), C.c_uint(1))

    def synchronize(self):
        _call("hipStreamSynchronize", self.handle)

    def close(self):
        _call("hipStreamDestroy", self.handle)


class Graph:
    """What `work` launches on a stream, captured."""

    def __init__(self, stream, work):
        self.stream, graph, self.handle = stream, C.c_void_p(), C.c_void_p()
        _call("hipStreamBeginCapture", stream.handle, C.c_int(2))  # relaxed
        try:
            work()
        finally:
            _call("hipStreamEndCapture", stream.handle, C.byref(graph))
        _call("hipGraphInstantiate", C.byref(self.handle), graph, None, None, C.c_size_t(0))
        _call("hipGraphDestroy", graph)

    def replay(self):
        _call("hipGraphLaunch", self.handle, self.stream.handle)

    def close(self):
        _call("hipGraphExecDestroy", self.handle)


def copy(to, source, stream):
    """All of `source` into `to`, device buffers of one size, on a stream."""
    _call("hipMemcpyAsync", to.ptr, source.ptr, C.c_size_t(source.nbytes), C.c_int(3),
          stream.handle)
