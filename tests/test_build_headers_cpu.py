"""Each translation unit's list of headers, by which stale objects are found, holds every header that the
unit includes, itself or through another one."""
import importlib.util
import os
import re

import pytest

from conftest import PKG_ROOT

spec = importlib.util.spec_from_file_location("k1_build_recipe", os.path.join(PKG_ROOT, "build.py"))
recipe = importlib.util.module_from_spec(spec)
spec.loader.exec_module(recipe)


def included(name, seen):
    for h in re.findall(r'#include "([^"]+\.cuh)"', open(os.path.join(recipe.CSRC, name)).read()):
        if h not in seen:
            seen.add(h)
            included(h, seen)
    return seen


@pytest.mark.parametrize("unit", sorted(recipe.CAPI_UNITS))
def test_headers_are_listed(unit):
    assert sorted(included(unit, set())) == sorted(recipe.CAPI_UNITS[unit])
