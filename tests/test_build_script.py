"""CPU: what csrc/build.sh compiles again.  The compiler is a stand-in that notes what it was asked to write."""
import os
import shutil
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_a_changed_build_script_compiles_every_object_again(tmp_path):
    """the script holds the compiler's flags: an object from before a change of them must not be linked"""
    src = tmp_path / "pkg" / "csrc"
    shutil.copytree(os.path.join(ROOT, "autognothi_amd", "csrc"), src)
    shutil.copytree(os.path.join(ROOT, "include"), tmp_path / "include")
    notes = tmp_path / "compiled"
    fake = tmp_path / "hipcc"
    fake.write_text(f"""#!/bin/bash
while [ $# -gt 0 ]; do case "$1" in -c) what="$2";; -o) out="$2";; esac; shift; done
echo built > "$out"
[ -z "$what" ] || echo "$what" >> {notes}
""")
    fake.chmod(0o755)

    def build():
        notes.write_text("")
        subprocess.run(["bash", str(src / "build.sh")], check=True, env={**os.environ, "HIPCC": str(fake)}, capture_output=True, timeout=60)
        return sorted(notes.read_text().split())

    def older(*paths):      # (by whole seconds, whatever the file system keeps)
        for p in paths:
            os.utime(p, (os.path.getatime(p) - 100, os.path.getmtime(p) - 100))

    older(*src.iterdir(), *(tmp_path / "include").iterdir())
    every = build()
    assert "logits.hip" in every and every.count("gemm_big.hip") == 2
    assert build() == []
    os.utime(src / "train.hip")
    older(*(src.parent / "lib").iterdir())
    assert build() == ["train.hip"]
    older(*(src.parent / "lib").iterdir())
    os.utime(src / "build.sh")
    assert build() == every
