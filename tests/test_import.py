"""What importing the package brings with it."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def python(code):
    subprocess.run([sys.executable, "-c", code], cwd=ROOT, check=True)


def test_the_package_and_its_bundle_writer_do_without_torch():
    python("import sys, lazyweights_amd, lazyweights_amd.bundle\n"
           "assert 'torch' not in sys.modules")


def test_attention_is_there_when_asked_for():
    python("import lazyweights_amd\n"
           "assert {'Batch', 'KvCache', 'Runtime'} <= set(dir(lazyweights_amd))\n"
           "from lazyweights_amd import Batch, KvCache\n"
           "from lazyweights_amd.attention import KvCache as same\n"
           "assert KvCache is same is lazyweights_amd.KvCache and Batch.__name__ == 'Batch'\n"
           "assert not hasattr(lazyweights_amd, 'Bach')\n")
