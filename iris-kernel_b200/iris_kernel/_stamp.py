"""What the bindings ``_ops.so`` were built for: they link torch's C++
libraries and this interpreter's ABI, so ``build.py`` builds them anew where
either is another one, and they are not loaded there before.  No imports of
the package: ``build.py`` loads this file by its path."""
import os
import sysconfig

PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_ops.stamp")


def present() -> str:
    import torch

    return f"torch {torch.__version__}, {sysconfig.get_config_var('SOABI')}"


def built(path: str = PATH) -> str | None:
    try:
        with open(path) as f:
            return f.read().strip()
    except OSError:
        return None
