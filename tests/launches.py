"""Which kernels a call of the library launches."""


def launched(handle, call):
    """(the call's result, the names of the kernels it launched)"""
    handle.set_kernel_timing(True)
    try:
        out = call()
        return out, [name for name, _ in handle.kernel_timings()]
    finally:
        handle.set_kernel_timing(False)
