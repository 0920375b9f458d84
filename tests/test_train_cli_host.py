"""Runs that the training commands refuse before anything is built, on the CPU."""
import pytest

from ofq_amd import train_cli


def test_cga_refuses_muon_before_anything_is_built():
    """FusedMuon cannot take CGA's element-wise freeze: cga.py says so at once, not after a forward and a backward pass."""
    for opt in ("muon", "Muon"):
        with pytest.raises(SystemExit, match="muon with cga.py"):
            train_cli.main(["--opt", opt], cga=True)
    args = train_cli.parse_args(["--opt", "muon"], False)
    train_cli.check_supported(args)
    train_cli.check_supported(train_cli.parse_args(["--opt", "adamw"], True), True)
