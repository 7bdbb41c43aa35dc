"""Arrivals at another block's barrier name the cluster's scope (the source says so; an arrival without
one orders nothing beyond its own block)."""
import re

import pytest

from inferx_b200.kernels import library


@pytest.mark.parametrize("path", library.sources() + library._headers(),
                         ids=lambda p: p.rsplit("/", 1)[-1])
def test_arrivals_at_other_blocks_are_of_cluster_scope(path):
    with open(path) as f:
        source = f.read()
    for form in re.findall(r"mbarrier\.arrive[\w.:]*", source):
        if "shared::cluster" in form:
            assert re.match(r"mbarrier\.arrive\.(release|relaxed)\.cluster\.", form), form
