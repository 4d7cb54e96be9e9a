import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (B200) and the built engine library")


def pytest_collection_modifyitems(items):
    """Tests of a binary that is built from the reference's sources come last where that binary is missing: they fail
    there, and a run that stops at its first failure has then run all others."""
    built = {"test_gpu_facade.py": os.path.join("yalama_b200", "host", "_build", "facade_chat"),
             "test_gpu_reference.py": os.path.join("oracle", "_ref", "ref_gpu_f16")}

    def missing(item):
        path = built.get(os.path.basename(str(item.fspath)))
        return path is not None and not os.path.exists(os.path.join(ROOT, path))

    items.sort(key=missing)
