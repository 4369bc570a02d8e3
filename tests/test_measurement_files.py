"""What keys the recorded counters to the machine code they were measured on: no GPU."""
from quantised_bayesian_nets_amd import build


def test_the_key_covers_sources_and_flags(monkeypatch, tmp_path):
    before = build.kernel_source_sha16()
    monkeypatch.setattr(build, "HIPCC_FLAGS", build.HIPCC_FLAGS[:-4])
    assert build.kernel_source_sha16() != before
    monkeypatch.undo()
    monkeypatch.setattr(build, "EXTRA", ["-DQBNN_STAMP"])
    assert build.kernel_source_sha16() != before
    monkeypatch.undo()
    changed = tmp_path / "qbnn_blocks.hip"
    changed.write_text("// another\n")
    monkeypatch.setattr(build, "SRC", [str(changed) if p.endswith("qbnn_blocks.hip") else p for p in build.SRC])
    assert build.kernel_source_sha16() != before
