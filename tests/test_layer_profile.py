"""profiles/layer.trace.tsv is of the committed kernels.

The script that takes it writes the digest of the sources it finds beside the figures.
A change to one of them makes this fail until the trace is taken again.
"""

import hashlib
import os

import __graft_entry__ as entry

PROFILE = os.path.join(entry.ROOT, "profiles", "layer.trace.tsv")
SOURCES = [*entry.LAYER_SOURCES, os.path.join(os.path.dirname(entry.SOURCE), "cfmoe_device.h")]


def test_layer_profile_is_of_the_current_sources():
    digest = hashlib.sha256()
    for path in SOURCES:
        with open(path, "rb") as f:
            digest.update(f.read())
    with open(PROFILE) as f:
        lines = [line for line in f if line.startswith("# sources ")]
    names = ", ".join(map(os.path.basename, SOURCES))
    assert lines == [f"# sources {names}, sha256 of them in a row: {digest.hexdigest()[:16]}\n"]
