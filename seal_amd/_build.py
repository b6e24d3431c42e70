"""Builds libsealfm.so (hipcc, gfx950 only) in-tree next to its sources: one object per source file (recompiled only
when the sha256 of that file, the headers and the flags changed -- not mtimes --, in parallel), then one link; the digest of everything
the library was built from is INSIDE it (`fmi_source_digest()`, a generated translation unit linked in last), and `stale()` compares that
with the sources present -- a sidecar file would pass when somebody replaces the binary alone (round 5's stamp)."""
import os
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(CSRC, "build")
LIB = os.path.join(CSRC, "libsealfm.so")
SOURCES = ["fmi_host.cpp", "fmi_evidence.cpp", "fmi_agg_pack.cpp", "fmi_sdsl.cpp", "fmi_kernels.hip", "fmi_aggregate.hip", "fmi_build_gpu.hip",
           "bart_kernels.hip", "hgemm_kernels.hip", "w4_kernels.hip", "kv8_kernels.hip", "sample_kernels.hip", "fmi_upload.hip"]
HEADERS = ["fmi_internal.h", "fmi_device.h", "fmi_agg.h", "nn_common.h", os.path.join("..", "..", "include", "sealfm.h"),
           os.path.join("..", "..", "include", "sealnn.h")]
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-ffp-contract=off", "-fPIC"]
# device code without packed fp32 instructions (v_pk_{add,mul,fma}_f32): hipcc -O3 forms them from ordinary float code, and some of their forms
# have given wrong results on gfx950 now and then.  (The host pass of a .hip file says that it does not know the feature: harmless.)
HIP_FLAGS = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def _hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found (ROCm toolchain required; this package targets gfx950 only)")


MARKER = b"SEALFM_SOURCE_DIGEST="          # in front of the 64 hex digits inside the binary (built_digest() finds it without loading the library)
OLD_STAMP = os.path.join(CSRC, "libsealfm.so.sha256")      # round 5's sidecar: removed when seen


def source_digest() -> str:
    """sha256 over every source, header and the flags: what libsealfm.so must have been built from.  (mtimes say nothing about a
    git-ignored binary that travels with a snapshot: a stale library with a fresh mtime would pass an mtime check.)"""
    import hashlib
    h = hashlib.sha256(" ".join(FLAGS + HIP_FLAGS).encode())
    for f in SOURCES + HEADERS:
        h.update(f.encode() + b"\0")
        with open(os.path.join(CSRC, f), "rb") as fh:
            h.update(fh.read())
    return h.hexdigest()


_digest_cache = {}


def built_digest() -> str:
    """the source digest embedded in libsealfm.so ("" if there is no library, or one built before the digest lived inside it); read from the
    file's bytes, so that a library built from other sources is recognised WITHOUT being loaded"""
    try:
        st = os.stat(LIB)
    except OSError:
        return ""
    key = (st.st_mtime_ns, st.st_size)
    if _digest_cache.get("key") != key:
        with open(LIB, "rb") as f:
            blob = f.read()
        at = blob.find(MARKER)
        hexd = blob[at + len(MARKER):at + len(MARKER) + 64].decode("ascii", "replace") if at >= 0 else ""
        _digest_cache.update(key=key, digest=hexd if len(hexd) == 64 and all(c in "0123456789abcdef" for c in hexd) else "")
    return _digest_cache["digest"]


def stale() -> bool:
    return not os.path.exists(LIB) or built_digest() != source_digest()


def _file_digest(path: str) -> str:
    import hashlib
    h = hashlib.sha256(" ".join(FLAGS + HIP_FLAGS).encode())
    for f in [path] + [os.path.join(CSRC, x) for x in HEADERS]:
        with open(f, "rb") as fh:
            h.update(fh.read())
    return h.hexdigest()


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not stale():
        if verbose:
            print("libsealfm.so is up to date with its sources (sha256 %s)" % built_digest()[:16], flush=True)
        return LIB
    os.makedirs(OBJ, exist_ok=True)
    hipcc = _hipcc()
    digest = source_digest()

    def compile_one(src: str) -> str:
        obj = os.path.join(OBJ, src + ".o")
        src_path = os.path.join(CSRC, src)
        want = _file_digest(src_path)
        try:
            with open(obj + ".sha256") as f:
                have = f.read().strip()
        except OSError:
            have = ""
        if force or not os.path.exists(obj) or have != want:
            cmd = [hipcc] + FLAGS + (HIP_FLAGS if src.endswith(".hip") else []) + ["-c", src_path, "-o", obj]
            if verbose:
                print(" ".join(cmd), flush=True)
            subprocess.check_call(cmd)
            with open(obj + ".sha256", "w") as f:
                f.write(want)
        return obj
    with ThreadPoolExecutor(max_workers=min(len(SOURCES), os.cpu_count() or 1)) as pool:
        objs = list(pool.map(compile_one, SOURCES))
    if os.path.exists(OLD_STAMP):
        os.remove(OLD_STAMP)
    # the digest, as one more translation unit (generated: it is a function of all the others)
    dsrc, dobj = os.path.join(OBJ, "fmi_source_digest.cpp"), os.path.join(OBJ, "fmi_source_digest.o")
    with open(dsrc, "w") as f:
        f.write('// generated by seal_amd/_build.py: the sha256 of the sources, headers and flags this library was built from\n'
                'static const char digest[] = "%s%s";\n'
                'extern "C" __attribute__((visibility("default"))) const char *fmi_source_digest(void) { return digest + %d; }\n'
                % (MARKER.decode(), digest, len(MARKER)))
    subprocess.check_call([hipcc, "--offload-arch=gfx950", "-O1", "-fPIC", "-c", dsrc, "-o", dobj])
    cmd = [hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB] + objs + [dobj]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    _digest_cache.clear()
    return LIB


if __name__ == "__main__":
    print(build(force=True, verbose=True))
