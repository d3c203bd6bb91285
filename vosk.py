"""`import vosk` for programs started in this folder: this module becomes the package in vosk-api_amd/."""
import importlib.machinery
import os

__path__ = [os.path.join(os.path.dirname(os.path.abspath(__file__)), "vosk-api_amd", "vosk")]
__file__ = os.path.join(__path__[0], "__init__.py")
__package__ = __name__
__spec__.submodule_search_locations = __path__
exec(importlib.machinery.SourceFileLoader(__name__, __file__).get_code(__name__))
