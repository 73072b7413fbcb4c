"""What bench.py takes for the source of a measured figure."""
import bench


def test_the_hash_of_a_source_is_of_it_and_of_the_headers_it_includes(tmp_path):
    files = {"a.hip": '#include "b.h"\n#include <other.h>\n#include "elsewhere.h"\n', "b.h": '#include "c.h"\n', "c.h": '#include "b.h"\n', "d.h": "x\n"}

    def hash_with(**changed):
        for name, text in {**files, **{k.replace("_", "."): v for k, v in changed.items()}}.items():
            (tmp_path / name).write_text(text)
        return bench.source_hash("a.hip", str(tmp_path))

    first = hash_with()
    assert hash_with(d_h="y\n", e_h="new\n") == first
    assert len({first, hash_with(a_hip=files["a.hip"] + "\n"), hash_with(b_h=files["b.h"] + "\n"), hash_with(c_h="\n")}) == 4


def test_every_measured_source_has_a_hash():
    import json
    import os
    with open(os.path.join(bench.ROOT, "profiles", "traffic.json")) as f:
        measured = json.load(f)
    for name, entry in measured.items():
        if isinstance(entry, dict) and "source" in entry:
            assert len(measured["source_sha256"][entry["source"]]) == len(bench.source_hash(entry["source"])) == 64, name
