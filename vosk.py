"""`import vosk` for programs started in this folder: the package in vosk-api_amd/."""
import importlib.util
import os
import sys


def _load():
    folder = os.path.join(os.path.dirname(os.path.abspath(__file__)), "vosk-api_amd", "vosk")
    spec = importlib.util.spec_from_file_location(__name__, os.path.join(folder, "__init__.py"),
                                                  submodule_search_locations=[folder])
    package = importlib.util.module_from_spec(spec)
    here = sys.modules[__name__]
    sys.modules[__name__] = package  # what the import statement returns
    try:
        spec.loader.exec_module(package)
    except BaseException:
        sys.modules[__name__] = here  # (the import statement takes it out)
        raise


_load()
