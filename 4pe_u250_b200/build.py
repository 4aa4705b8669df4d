"""Builds the native parts of the package in-tree.

  libi4d.so        the CUDA decode library (sm_100a) behind include/i4d.h
  libi4d_synth.so  seeded synthetic model images in the reference format
  _i4d_torch.so    torch binding of the long-context operators
  i4d_decode       C++ host program over libi4d (replaces decode_host)
  csrc/gen/*       build-time tables (expf constants and exceptions)

Run as ``python -m`` or through ``__graft_entry__.build()``.  The expf
exception table is measured against this machine's C library once and
reused while its inputs are unchanged.
"""
import hashlib
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
GEN = os.path.join(CSRC, "gen")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def _run(cmd, cwd=None):
    print("+", " ".join(cmd), flush=True)
    subprocess.run(cmd, check=True, cwd=cwd)


def _digest(paths):
    h = hashlib.sha256()
    for p in paths:
        with open(p, "rb") as f:
            h.update(f.read())
    return h.hexdigest()


def _newer(target, sources):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(s) > t for s in sources)


def build_expf_tables():
    os.makedirs(GEN, exist_ok=True)
    consts = os.path.join(GEN, "expf_consts.h")
    gen_py = os.path.join(CSRC, "gen_expf_consts.py")
    if _newer(consts, [gen_py]):
        _run([sys.executable, gen_py, consts])
    impl = os.path.join(CSRC, "i4d_expf_impl.h")
    tool_src = os.path.join(CSRC, "gen_expf_table.c")
    table = os.path.join(GEN, "expf_fix_table.c")
    stamp = os.path.join(GEN, "expf_fix_table.sha256")
    key = _digest([consts, impl, tool_src])
    if os.path.exists(table) and os.path.exists(stamp) and open(stamp).read().strip() == key:
        return table
    tool = os.path.join(GEN, "gen_expf_table")
    _run(["gcc", "-O2", "-mfma", "-ffp-contract=off", "-fopenmp", "-I", CSRC, tool_src, "-o", tool, "-lm"])
    _run([tool, table])
    with open(stamp, "w") as f:
        f.write(key + "\n")
    return table


def build_synth():
    src = os.path.join(CSRC, "synth.c")
    out = os.path.join(HERE, "libi4d_synth.so")
    if _newer(out, [src]):
        _run(["gcc", "-O2", "-std=c11", "-fopenmp", "-fPIC", "-shared", src, "-o", out, "-lm"])
    return out


def build_i4d():
    table = build_expf_tables()
    srcs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh", ".h"))]
    srcs.append(os.path.join(ROOT, "include", "i4d.h"))
    out = os.path.join(HERE, "libi4d.so")
    if not _newer(out, srcs + [table]):
        return out
    obj_dir = os.path.join(ROOT, "_build")
    os.makedirs(obj_dir, exist_ok=True)
    tab_obj = os.path.join(obj_dir, "expf_fix_table.o")
    headers = [s for s in srcs if not s.endswith(".cu")]
    # The decode path rounds every product and sum by itself; the serving
    # operators state their rounding order where it matters.
    units = [("i4d.cu", ["-fmad=false"]), ("i4d_ops.cu", [])]
    running, objs = [], []
    for name, flags in units:
        src = os.path.join(CSRC, name)
        obj = os.path.join(obj_dir, name[:-3] + ".o")
        objs.append(obj)
        if _newer(obj, headers + [src]):
            cmd = [NVCC, *ARCH, "-lineinfo", "-O3", "-std=c++17", *flags, "-Xptxas", "-v", "-Xcompiler", "-fPIC",
                   "-I", os.path.join(ROOT, "include"), "-I", CSRC, "-c", src, "-o", obj]
            print("+", " ".join(cmd), flush=True)
            running.append((cmd, subprocess.Popen(cmd)))
    failed = [cmd for cmd, p in running if p.wait() != 0]
    if failed:
        raise subprocess.CalledProcessError(1, failed[0])
    _run(["gcc", "-O1", "-fPIC", "-c", table, "-o", tab_obj])
    _run([NVCC, *ARCH, "-shared", "-o", out, *objs, tab_obj])
    return out


def build_torch():
    """The torch binding of the long-context operators, against this interpreter's torch."""
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths
    src = os.path.join(CSRC, "i4d_torch.cpp")
    out = os.path.join(HERE, "_i4d_torch.so")
    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    if _newer(out, [src, os.path.join(ROOT, "include", "i4d.h"), os.path.join(HERE, "libi4d.so")]):
        inc = [sysconfig.get_path("include"), os.path.join(os.path.dirname(os.path.dirname(NVCC)), "include"), *include_paths()]
        _run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
              f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I", os.path.join(ROOT, "include"),
              *[f"-I{i}" for i in inc], src, "-o", out, "-L" + HERE, "-l:libi4d.so", "-Wl,-rpath,$ORIGIN", "-L" + lib,
              "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda"])
    return out


def build_host():
    src = os.path.join(CSRC, "host", "i4d_decode.cpp")
    out = os.path.join(HERE, "i4d_decode")
    lib = os.path.join(HERE, "libi4d.so")
    if _newer(out, [src, lib, os.path.join(ROOT, "include", "i4d.h")]):
        _run(["g++", "-O2", "-std=c++17", "-I", os.path.join(ROOT, "include"), src, "-o", out,
              "-L" + HERE, "-l:libi4d.so", "-Wl,-rpath,$ORIGIN"])
    return out


def build_oracle():
    """The C restatement always; the reference emulator (oracle/_ref) only
    where I4D_REF_ROOT names a reference tree that holds its source."""
    _run(["make", "-s", "-C", os.path.join(ROOT, "oracle"), "oracle"])
    ref_root = os.environ.get("I4D_REF_ROOT")
    source = os.path.join("software_sim", "llama2_decoder_sw_emulator.cpp")
    if ref_root and os.path.isfile(os.path.join(ref_root, source)):
        _run(["make", "-s", "-C", os.path.join(ROOT, "oracle"), "ref", "REF_ROOT=" + ref_root])


def main():
    build_synth()
    build_i4d()
    build_host()
    build_oracle()
    # Last, and only where there is a torch to bind to; a call of the operators
    # from Python says that the binding is missing.
    try:
        import torch  # noqa: F401
    except ImportError:
        print("no torch: the binding of the long-context operators is not built", flush=True)
        return
    build_torch()


if __name__ == "__main__":
    main()
