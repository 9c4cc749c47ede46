"""Every compiler call that makes GPU code is given the same flags, and a change of the Makefile reaches every object."""
import glob
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NO_PACKED = "-Xclang -target-feature -Xclang -packed-fp32-ops"


def test_no_gpu_code_is_compiled_with_packed_fp32_instructions():
    lines = []
    for path in [os.path.join(ROOT, "rag_amd/csrc/Makefile")] + glob.glob(os.path.join(ROOT, "scripts/*.sh")):
        for line in open(path).read().replace("\\\n", " ").splitlines():
            if re.search(r"(^|\s)-c\s+\S*(\.hip|\$f)", line) and "hipcc" in line or line.startswith("CXXFLAGS"):
                lines.append((path, line))
    assert len(lines) >= 5                                  # the Makefile's flags and four scripts
    for path, line in lines:
        assert NO_PACKED in line, (path, line)


def test_a_change_of_the_makefile_compiles_everything_again():
    say = subprocess.run(["make", "-n", "-W", "Makefile", "-C", os.path.join(ROOT, "rag_amd/csrc")], capture_output=True, text=True, check=True).stdout
    for source in glob.glob(os.path.join(ROOT, "rag_amd/csrc/*.hip")):
        assert "-c %s " % os.path.basename(source) in say, source
