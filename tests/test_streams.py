"""-m "not gpu": what the sources may ask of HIP streams."""
import glob
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_stream_has_the_default_priority():
    """Work on streams of different priorities has hung the device for good: nothing in the package, the bench or the tools asks for another one."""
    for f in glob.glob(os.path.join(ROOT, "deft_amd", "**", "*.py"), recursive=True) + glob.glob(os.path.join(ROOT, "deft_amd", "csrc", "*")) + \
            glob.glob(os.path.join(ROOT, "tools", "**", "*.py"), recursive=True) + [os.path.join(ROOT, "bench.py"), os.path.join(ROOT, "run_stream.py"), os.path.join(ROOT, "detector.py")]:
        src = open(f).read()
        assert not re.search(r"Stream\([^)]*priority|StreamCreateWithPriority|is_high_priority_stream", src), f
