"""HIP graphs over the runtime's C interface, for tests that capture calls."""
import ctypes as C


class Graph:
    """The work that record() queues on the context's stream, captured."""

    def __init__(self, ctx, record):
        self.hip = C.CDLL("libamdhip64.so")
        for f, args in (("hipStreamBeginCapture", [C.c_void_p, C.c_int]), ("hipStreamEndCapture", [C.c_void_p, C.POINTER(C.c_void_p)]),
                        ("hipGraphInstantiate", [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t]),
                        ("hipGraphLaunch", [C.c_void_p, C.c_void_p]), ("hipGraphDestroy", [C.c_void_p]), ("hipGraphExecDestroy", [C.c_void_p])):
            getattr(self.hip, f).argtypes = args
        self.ctx, self.graph, self.exe = ctx, C.c_void_p(), C.c_void_p()
        ctx.sync()
        assert self.hip.hipStreamBeginCapture(ctx.stream(), 1) == 0        # 1: this thread's calls only
        try:
            record()
        finally:
            assert self.hip.hipStreamEndCapture(ctx.stream(), C.byref(self.graph)) == 0
        assert self.hip.hipGraphInstantiate(C.byref(self.exe), self.graph, None, None, 0) == 0

    def replay(self):
        assert self.hip.hipGraphLaunch(self.exe, self.ctx.stream()) == 0

    def close(self):
        self.ctx.sync()
        self.hip.hipGraphExecDestroy(self.exe)
        self.hip.hipGraphDestroy(self.graph)
