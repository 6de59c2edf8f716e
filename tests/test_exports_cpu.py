"""What the packages import for their users, a star import gives them too."""
import importlib
import inspect

import pytest


@pytest.mark.parametrize("name", ["mamba_amd.ops", "mamba_amd.modules", "mamba_amd.models"])
def test_star_import_gives_every_name(name):
    package = importlib.import_module(name)
    public = {n for n, v in vars(package).items() if not n.startswith("_") and not inspect.ismodule(v)}
    assert public == set(package.__all__) and len(package.__all__) == len(public)
    got = {}
    exec(f"from {name} import *", got)
    assert public <= set(got)
