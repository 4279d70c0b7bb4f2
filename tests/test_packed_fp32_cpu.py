"""No GPU code here holds packed fp32 arithmetic: none is written by hand, and every line that builds GPU code tells the compiler to form none."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FLAG = "-Xclang -target-feature -Xclang -packed-fp32-ops"
PACKED = re.compile(r"v_pk_\w+_f32")


def files(*endings):
    for folder in ("vidchapters_amd", "include", "tools"):
        for base, dirs, names in os.walk(os.path.join(ROOT, folder)):
            dirs[:] = [d for d in dirs if d not in ("build", "__pycache__")]
            yield from (os.path.join(base, n) for n in names if n.endswith(endings))


def test_no_packed_fp32_by_hand():
    seen = 0
    for path in files(".hip", ".h", ".inc", ".py"):
        seen += 1
        with open(path) as f:
            assert not PACKED.search(f.read()), path
    assert seen > 20


def test_every_build_of_gpu_code_has_the_flag():
    seen = 0
    for path in files(".sh"):
        with open(path) as f:
            text = f.read()
        if "hipcc" not in text or "-c " not in text:
            continue
        seen += 1
        assert "FLAGS=" in text and FLAG in text, path
        for line in text.splitlines():
            if re.search(r"(\$HIPCC|bin/hipcc) .*\.hip", line):
                assert "$FLAGS" in line, (path, line)
    assert seen >= 5
    for path in files(".hip"):
        with open(path) as f:
            for line in f:
                if "build: hipcc" in line:
                    assert FLAG in line, (path, line)
