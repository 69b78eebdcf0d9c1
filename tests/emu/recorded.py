"""Which kernels libfg_mi355.so launches for a call, without running any: the library's host code as built, against the HIP
stand-in (hip_shim.cpp), in a process of its own.

    python tests/emu/recorded.py LIB SHIM_DIR < calls.json > answers.json

calls: [entry point, struct bytes as hex] in a list; the struct goes in by reference, the stream is NULL.  Answers: one
[return code, fg_last_error(), [[kernel, grid, block, hex], ...]] for each; hex: as many bytes of the kernel's first argument as the
struct has (kernels of these entry points take a copy of it in front of what they add)."""
import ctypes
import json
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from device import _LAUNCH_CB, _SYMBOL_CB, build_shim  # noqa: E402


def main(lib_path, shim_dir):
    launches, size = [], 0

    def on_launch(name, grid, block, args, shmem, stream):
        launches.append([name.decode(), list(grid[:3]), list(block[:3]), ctypes.string_at(args[0], size).hex()])
        return 0

    shim = ctypes.CDLL(build_shim(shim_dir), mode=ctypes.RTLD_GLOBAL)
    callbacks = _LAUNCH_CB(on_launch), _SYMBOL_CB(lambda name, n: 0)
    shim.shim_set_callbacks(*callbacks)
    lib = ctypes.CDLL(lib_path)
    lib.fg_last_error.restype = ctypes.c_char_p
    assert shim.shim_num_functions() > 0, "the real HIP runtime was bound"
    answers = []
    for name, struct in json.load(sys.stdin):
        launches.clear()
        size = len(struct) // 2
        data = ctypes.create_string_buffer(bytes.fromhex(struct))
        rc = getattr(lib, name)(data, None)
        answers.append([rc, (lib.fg_last_error() or b"").decode() if rc else "", list(launches)])
    json.dump(answers, sys.stdout)


if __name__ == "__main__":
    main(*sys.argv[1:3])
