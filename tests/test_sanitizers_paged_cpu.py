"""Host code of the paged 4-bit cache in service under
AddressSanitizer and UndefinedBehaviorSanitizer, on the CPU: its entry points and
launchers, host pass instrumented, driven through rejections, size queries and calls
that have nothing to do (sanitize_paged_main.cpp; no call reaches a kernel launch)."""
from __future__ import annotations

from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

from test_sanitizers_cpu import CSRC, ENV, HERE, HOST_SAN, ROOT, _hipcc, _run

SOURCES = ["capi_paged.cpp", "kv4.hip", "kv4_pages.hip", "kv4_chunks.hip", "kv4_unpacked.hip"]


def test_paged_host_code_under_sanitizers(tmp_path):
    hipcc = _hipcc()
    flags = ["-std=c++17", "-O1", "-g", "--offload-arch=gfx950", "-fPIC",
             "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
             f"-I{ROOT / 'include'}", *HOST_SAN]

    def compile_one(src):
        obj = tmp_path / (src.stem + ".o")
        return obj, _run([hipcc, "-x", "hip", *flags, "-c", str(src), "-o", str(obj)])

    sources = [CSRC / s for s in SOURCES] + [HERE / "sanitize_paged_main.cpp"]
    with ThreadPoolExecutor(max_workers=len(sources)) as ex:
        results = list(ex.map(compile_one, sources))
    for _, (rc, out) in results:
        assert rc == 0, out[-3000:]
    exe = tmp_path / "sanitize_paged"
    rc, res = _run([hipcc, "-print-resource-dir"])
    assert rc == 0, res
    rt = Path(res.strip().splitlines()[-1]) / "lib" / "linux"
    rc, out = _run([hipcc, "--offload-arch=gfx950", *HOST_SAN, "-shared-libsan", "-o", str(exe),
                    *(str(o) for o, _ in results), f"-Wl,-rpath,{rt}"])
    assert rc == 0, out[-3000:]
    rc, out = _run([str(exe)], env=ENV)
    assert rc == 0 and "OK" in out, out[-4000:]
