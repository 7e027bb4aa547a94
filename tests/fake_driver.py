"""Programs run over fake_cuda.c: what they enqueue, and what of it is ordered."""

import os
import subprocess
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
CUDA = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda"))


def run(program, folder, slow=None, slow_compile=None, before=""):
    """Runs `program` (Python text, with `api` and `np` in hand) in a process
    whose CUDA driver and NVRTC are the stand-in; its output, and the log's
    lines, split. `slow`: a kernel each of whose launches takes 0.4 s on the
    host (or cuEventRecord); `slow_compile`: text of sources that take a second to compile;
    `before` runs before the import of the api."""
    library, log = folder / "libcuda.so.1", folder / "log"
    if not library.exists():
        (folder / "libnvrtc.so.12").symlink_to(library)
        subprocess.run(["gcc", "-O1", "-w", "-shared", "-fPIC", f"-I{CUDA / 'include'}", str(HERE / "fake_cuda.c"),
                        "-o", str(library), "-lpthread"], check=True)
    env = dict(os.environ, LD_LIBRARY_PATH=f"{folder}:{os.environ.get('LD_LIBRARY_PATH', '')}",
               FAKE_CUDA_LOG=str(log), PYTHONPATH=str(HERE.parent), **{k: v for k, v in
               (("FAKE_CUDA_SLOW", slow), ("FAKE_CUDA_SLOW_COMPILE", slow_compile)) if v})
    env.pop("PORCH_B200_CACHE_DIR", None)
    head = before + "import threading, time, os\nimport numpy as np\nfrom porch_b200 import api\n"
    done = subprocess.run([sys.executable, "-c", head + program], env=env, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr
    return done.stdout, [line.split() for line in log.read_text().splitlines()]


def unordered(log, conflicts):
    """Pairs of launches, in the order of the log, for which conflicts(first,
    second) holds (both kernels' names) and which no stream, event or host wait
    puts one behind the other."""
    streams, events, threads, names, bad = {}, {}, {}, [], []
    for thread, what, *rest in log:
        host = threads.setdefault(thread, set())
        if what == "record":
            events[rest[1]] = set(streams.get(rest[0], ()))
        elif what == "wait":
            streams.setdefault(rest[0], set()).update(events.get(rest[1], ()))
        elif what == "sync":
            host |= streams.get(rest[0], set())
        elif what == "launch":
            before = streams.setdefault(rest[0], set())
            before |= host
            bad += [(names[i], rest[1]) for i in range(len(names)) if i not in before and conflicts(names[i], rest[1])]
            before.add(len(names))
            names.append(rest[1])
    return bad
