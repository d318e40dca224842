"""Build the MI355X HIP library in-tree: ur3e_amd/_lib/libur3e_amd.so (gfx950).

Before compiling, the static dof tree of assets/main.model.json is emitted as constexpr
tables (csrc/gen_main_tree.h): the compact-tier kernel specialised for that model folds
every tree test at compile time.  The host only picks that kernel when the loaded model's
tree matches the tables (ur3e_batch_create compares them)."""
import json
import os
import subprocess
import time

HERE = os.path.dirname(os.path.abspath(__file__))
SRC = os.path.join(HERE, "csrc", "ur3e_batch.hip")
SRC_VN = os.path.join(HERE, "csrc", "ur3e_vecnorm.hip")
SRC_PL = os.path.join(HERE, "csrc", "ur3e_policy.hip")  # the operators of ur3e_amd/rl/ops.py
SRC_PL_TORCH = os.path.join(HERE, "csrc", "ur3e_policy_torch.cpp")  # their torch binding, a library of its own
SRC_MJCF = os.path.join(HERE, "csrc", "ur3e_mjcf.cpp")  # host only: the MJCF / YAML entry points
SRC_GATHER = os.path.join(HERE, "csrc", "ur3e_gather.cpp")  # host only: the RCCL gather entry point
DEPS = [SRC, SRC_VN, SRC_PL, SRC_MJCF, SRC_GATHER, os.path.join(HERE, "..", "include", "ur3e_vecnorm.h"),
        os.path.join(HERE, "..", "include", "ur3e_policy.h"), os.path.join(HERE, "csrc", "ur3e_engine.h"), os.path.join(HERE, "csrc", "ur3e_wave.h"), os.path.join(HERE, "csrc", "ur3e_wave_r.h"),
        os.path.join(HERE, "csrc", "detmath.h"), os.path.join(HERE, "csrc", "gen_main_tree.h"),
        os.path.join(HERE, "csrc", "convex.h"), os.path.join(HERE, "csrc", "ur3e_cvx_wave.h"),
        os.path.join(HERE, "..", "include", "ur3e_model.h"), os.path.join(HERE, "..", "include", "ur3e_batch.h")]
GEN = os.path.join(HERE, "csrc", "gen_main_tree.h")
MAIN_JSON = os.path.join(HERE, "assets", "main.model.json")
LIB = os.path.join(HERE, "_lib", "libur3e_amd.so")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-ffp-contract=off", "-fPIC", "-shared",
         # machine LICM hoisted loop-invariant constants and addresses out of the substep and queue loops,
         # keeping them live across the whole step: SGPR spills into VGPR lanes, 256 VGPRs and scratch.
         # Without it every step kernel is scratch-free at 207-212 VGPRs (ur3e_batch.hip kernels)
         "-mllvm", "-disable-machine-licm",
         "-Wno-unused-result"]
# the policy operators are float kernels of their own: contraction to FMAs and loop-invariant motion as the
# compiler chooses, but no packed float instructions (some of their forms have given wrong results on gfx950)
FLAGS_PL = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Xclang", "-target-feature", "-Xclang",
            "-packed-fp32-ops", "-Wno-unused-result"]


def gen_main_tree() -> str:
    """Emit the dof-ancestor masks and body parents of main.xml as constexpr tables (rewritten only on
    change)."""
    with open(MAIN_JSON) as f:
        md = json.load(f)
    nv = md["nv"]
    par = md["dof_parentid"][:nv]
    masks = []
    for i in range(nv):
        mask, j = 0, par[i]
        while j >= 0:
            mask |= 1 << j
            j = par[j]
        masks.append(mask)
    nb = md["nbody"]
    bpar = md["body_parentid"][:nb]
    bdn = md["body_dofnum"][:nb]
    bja = md["body_jntadr"][:nb]
    jtype = md["jnt_type"]
    # several-dof bodies: free joints hanging off the world, without children
    cols = int(all(bpar[i] == 0 and i not in bpar and md["body_jntnum"][i] == 1 and jtype[bja[i]] == 0
                   for i in range(1, nb) if bdn[i] > 1))
    split = 0
    for cand in range(1, nv):
        lo_ok = all((masks[i] >> cand) == 0 for i in range(cand))          # dofs < cand: ancestors < cand
        hi_ok = all((masks[i] & ((1 << cand) - 1)) == 0 for i in range(cand, nv))  # dofs >= cand: none < cand
        # the kernel's interleaved block Cholesky needs the trailing tree no larger than the leading one
        if lo_ok and hi_ok and nv - cand <= cand:
            split = cand
    txt = ("/* generated by ur3e_amd/_build.py from assets/main.model.json -- do not edit */\n"
           "#ifndef UR3E_GEN_MAIN_TREE_H\n#define UR3E_GEN_MAIN_TREE_H\n"
           f"#define UR3E_MAIN_NV {nv}\n"
           "/* bit j of mask i: dof j is a proper ancestor of dof i (KPlan.dof_anc_mask) */\n"
           f"static constexpr unsigned int ur3e_main_dof_anc_mask[{nv}] = {{"
           + ", ".join(f"0x{x:x}u" for x in masks) + "};\n"
           "/* first dof of the last dof tree when the dofs split into two trees [0, S) and [S, nv) with no\n"
           "   ancestor across (0: no such split): the mass matrix is block diagonal over them */\n"
           f"#define UR3E_MAIN_SPLIT {split}\n"
           "/* body tree: subtree sums with compile-time parents (r_subtree_sum_cols) */\n"
           f"#define UR3E_MAIN_NB {nb}\n"
           f"static constexpr int ur3e_main_body_parent[{nb}] = {{"
           + ", ".join(str(x) for x in bpar) + "};\n"
           f"static constexpr int ur3e_main_body_dofnum[{nb}] = {{"
           + ", ".join(str(x) for x in bdn) + "};\n"
           f"static constexpr int ur3e_main_body_jntadr[{nb}] = {{"
           + ", ".join(str(x) for x in bja) + "};\n"
           "/* 1: every body with several dofs is a free joint hanging off the world without children, so the\n"
           "   position, velocity and acceleration chains run with the components across lanes */\n"
           f"#define UR3E_MAIN_BODY_COLS {cols}\n#endif\n")
    old = open(GEN).read() if os.path.exists(GEN) else None
    if old != txt:
        with open(GEN, "w") as f:
            f.write(txt)
    return GEN


GEN_PY = os.path.join(HERE, "csrc", "gen_pyconfig.h")


def gen_pyconfig() -> str:
    """Emit the building interpreter's libpython (path and soname) for the C ABI's embedded compiler
    (csrc/ur3e_mjcf.cpp: the first candidates it dlopens when UR3E_LIBPYTHON is unset), rewritten only on
    change.  A statically linked interpreter has no shared libpython: both stay empty there."""
    import sysconfig
    libdir = sysconfig.get_config_var("LIBDIR") or ""
    soname = sysconfig.get_config_var("INSTSONAME") or ""
    if ".so" not in soname:  # a static libpython (.a): nothing to dlopen
        soname = ""
    path = os.path.join(libdir, soname) if (libdir and soname) else ""
    if path and not os.path.exists(path):
        path = ""

    def c(x):
        return '"' + x.replace("\\", "\\\\").replace('"', '\\"') + '"'
    txt = ("/* generated by ur3e_amd/_build.py from the building interpreter's sysconfig -- do not edit */\n"
           "#ifndef UR3E_GEN_PYCONFIG_H\n#define UR3E_GEN_PYCONFIG_H\n"
           f"#define UR3E_BUILD_LIBPYTHON {c(path)}\n"
           f"#define UR3E_BUILD_LIBPYTHON_SONAME {c(soname)}\n#endif\n")
    old = open(GEN_PY).read() if os.path.exists(GEN_PY) else None
    if old != txt:
        with open(GEN_PY, "w") as f:
            f.write(txt)
    return GEN_PY


# diagnostic variant built beside the product library: the queue-unit trace (tools/queue_trace.py,
# tests/test_gpu_queue.py) -- unit stamps stored from lane 0 inside the queue kernel's loop
TRACE_LIB = os.path.join(HERE, "_lib", "libur3e_amd_trace.so")
TRACE_DEFS = ["-DUR3E_WAVE_TRACE", "-DUR3E_TRACE_LANE0"]
OBJ = os.path.join(HERE, "_lib", "obj")
# each source compiles to its own object (only a changed source and what includes it recompile; the step
# kernels' translation unit takes minutes, the host-only entry points seconds), then the library links.  Each
# compile writes a depfile (hipcc -MD) next to its object, so an object is stale when any file it actually
# included is newer; before the first build (no depfile yet) every header of the tree counts.
HEADERS = [d for d in DEPS if d.endswith(".h")] + [GEN_PY]
SOURCES = [SRC, SRC_VN, SRC_PL, SRC_MJCF, SRC_GATHER]


def _newer(out: str, deps) -> bool:
    if not os.path.exists(out):
        return True
    t = os.path.getmtime(out)
    return any(not os.path.exists(d) or os.path.getmtime(d) > t for d in deps)


def _depfile_deps(dep: str):
    """the files a compile read (its depfile's prerequisites), or None when there is no depfile"""
    if not os.path.exists(dep):
        return None
    with open(dep) as f:
        txt = f.read().replace("\\\n", " ")
    _, _, rest = txt.partition(":")
    root = os.path.dirname(HERE)
    # the tree's own files only (system and ROCm headers change with the image, not with a commit)
    return [d for d in rest.split() if os.path.abspath(d).startswith(root)]


def _stale(lib: str) -> bool:
    return _newer(lib, DEPS)


def _objects(defs, tag, force, verbose):
    """(object paths, compile jobs) for one library variant; the step kernels' object is per variant"""
    objs, jobs = [], []
    for src in SOURCES:
        var = tag if src == SRC else ""
        obj = os.path.join(OBJ, os.path.basename(src) + var + ".o")
        dep = obj + ".d"
        objs.append(obj)
        deps = _depfile_deps(dep)
        if force or _newer(obj, [src] + (deps if deps is not None else HEADERS)):
            flags = FLAGS_PL if src == SRC_PL else [f for f in FLAGS if f != "-shared"]
            cmd = ([HIPCC] + flags + (defs if src == SRC else [])
                   + ["-MD", "-MF", dep, "-c", "-o", obj, src])
            if verbose:
                print(" ".join(cmd))
            jobs.append((cmd, obj))
    return objs, jobs


# the policy operators' torch binding: host code against this interpreter's torch, linked to the product library
# beside it
TORCH_LIB = os.path.join(HERE, "_lib", "ur3e_policy_torch.so")


def _torch_cmd():
    import sysconfig

    import torch
    from torch.utils import cpp_extension as ce
    lib = ce.library_paths()[0]
    return (["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
             "-DTORCH_EXTENSION_NAME=ur3e_policy_torch",
             f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
            + [f"-I{p}" for p in ce.include_paths()] + [f"-I{sysconfig.get_paths()['include']}", "-I/opt/rocm/include"]
            + ["-MD", "-MF", os.path.join(OBJ, "ur3e_policy_torch.d"), SRC_PL_TORCH, "-o", TORCH_LIB,
               f"-L{os.path.dirname(LIB)}", "-lur3e_amd", "-Wl,-rpath,$ORIGIN", f"-L{lib}", "-ltorch_python", "-ltorch",
               "-ltorch_cpu", "-ltorch_hip", "-lc10", "-lc10_hip"])


def _build_torch(force, verbose):
    try:
        import torch
    except ImportError:
        # the C library serves its C users without; ur3e_amd.rl.ops raises
        print("torch is not importable: the policy operators' torch binding (ur3e_policy_torch.so) is not built")
        return
    cmd = _torch_cmd()
    # what it was built with: another torch, or another command, is another binding
    stamp = os.path.join(OBJ, "ur3e_policy_torch.cmd")
    made_by = "\n".join([torch.__version__, *cmd])
    try:
        with open(stamp) as f:
            same = f.read() == made_by
    except OSError:
        same = False
    deps = _depfile_deps(os.path.join(OBJ, "ur3e_policy_torch.d"))
    if force or not same or _newer(TORCH_LIB, [SRC_PL_TORCH] + (deps if deps is not None else HEADERS)):
        if verbose:
            print(" ".join(cmd))
        t0 = time.time()
        subprocess.run(cmd, check=True)
        os.utime(TORCH_LIB, (t0, t0))
        with open(stamp, "w") as f:
            f.write(made_by)


def build(force: bool = False, verbose: bool = False, trace: bool = False) -> str:
    """Build the product library (and, with trace=True, the trace variant) when a source is newer.
    Objects compile in parallel; a library relinks when one of its objects changed."""
    os.makedirs(OBJ, exist_ok=True)
    gen_main_tree()
    gen_pyconfig()
    plans, jobs, seen = [], [], set()
    for lib, defs, tag, want in ((LIB, [], "", True), (TRACE_LIB, TRACE_DEFS, ".trace", trace)):
        if not want:
            continue
        objs, js = _objects(defs, tag, force, verbose)
        plans.append((lib, objs))
        for cmd, obj in js:
            if obj not in seen:
                seen.add(obj)
                jobs.append((cmd, obj, time.time(), subprocess.Popen(cmd)))
    for cmd, obj, t0, pr in jobs:
        if pr.wait() != 0:
            raise subprocess.CalledProcessError(pr.returncode, cmd)
        # the object is as old as the sources the compile read: a source edited while it ran stays newer
        # than the object, so the next build recompiles it
        os.utime(obj, (t0, t0))
    for lib, objs in plans:
        if force or _newer(lib, objs):
            cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", lib] + objs + ["-ldl"]
            if verbose:
                print(" ".join(cmd))
            subprocess.run(cmd, check=True)
    _build_torch(force, verbose)
    return LIB


if __name__ == "__main__":
    build(force=True, verbose=True, trace=True)
