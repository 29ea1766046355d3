"""The command line's options for feed-forwards in 8 bits: what they refuse and hand on, and a run of them on the GPU."""
import json
import os
import subprocess
import sys

import pytest

import harness as H  # noqa: F401  (path setup)
from tiny_configs import TINY_A

from lastengine_b200.cli import main


def test_8_bits_beside_32_are_refused_in_words(tmp_path):
    p = tmp_path / "config.json"
    p.write_text(json.dumps(TINY_A))
    with pytest.raises(SystemExit, match="lastengine generate: .*bfloat16 engine, not float32"):
        main(["generate", "--config", str(p), "--prompt-ids", "1,2,3", "--dtype", "float32", "--ffn-dtype", "e4m3"])


def test_the_comparing_tools_take_the_option(monkeypatch):
    """dense-cmp puts it on the path under test alone, replay hands it on."""
    from lastengine_b200 import cli
    for command in (["dense-cmp", "dir", "1,2"], ["replay", "--model", "m", "--dtype", "bfloat16", "--out", "o", "--max-tokens", "64"]):
        assert cli.build_parser().parse_args(command).ffn_dtype is None
        assert cli.build_parser().parse_args(command + ["--ffn-dtype", "e4m3"]).ffn_dtype == "e4m3"
    asked = []

    class Enough(Exception):
        pass

    def engine(path, dtype, ctx, ffn_dtype=None):
        asked.append((dtype, ffn_dtype))
        if len(asked) == 2:
            raise Enough
    monkeypatch.setattr(cli, "_engine", engine)
    with pytest.raises(Enough):
        main(["dense-cmp", "dir", "1,2", "--ffn-dtype", "e4m3"])
    assert asked == [("float32", None), ("bfloat16", "e4m3")]
    ran = []
    monkeypatch.setattr(cli.os, "execv", lambda exe, args: ran.append(args))
    main(["replay", "--model", "m", "--dtype", "bfloat16", "--out", "o", "--max-tokens", "64", "--ffn-dtype", "e4m3"])
    main(["replay", "--model", "m", "--dtype", "bfloat16", "--out", "o", "--max-tokens", "64"])
    assert ran[0][-2:] == ["--ffn-dtype", "e4m3"] and "--ffn-dtype" not in ran[1]


def test_trace_run_refuses_8_bits_beside_32():
    p = subprocess.run([sys.executable, os.path.join(H.ROOT, "bin", "trace_run"), "--model", "m", "--dtype", "float32", "--out", "o", "--max-tokens", "64",
                        "--ffn-dtype", "e4m3"], capture_output=True, text=True, timeout=120)
    assert p.returncode == 2 and "--ffn-dtype e4m3 goes with --dtype bfloat16" in p.stderr


@pytest.mark.gpu
def test_the_comparing_tools_run_in_8_bits(tmp_path, capsys):
    d = H.make_model_dir(TINY_A, 0, str(tmp_path / "m"))
    assert main(["dense-cmp", d, "1,2,3", "6", "--ffn-dtype", "e4m3"]) == 0
    assert "/6 argmax agree" in capsys.readouterr().out
    step = json.dumps({"step": 0, "entries": [{"id": "a", "tokens": [5, 17, 3], "want": [0, 2]}], "end": ["a"]})
    got = {}
    for ffn in ([], ["--ffn-dtype", "e4m3"]):
        out = tmp_path / f"out{len(ffn)}"
        p = subprocess.run([sys.executable, os.path.join(H.ROOT, "bin", "trace_run"), "--model", d, "--dtype", "bfloat16", "--out", str(out), "--max-tokens", "64", *ffn],
                           input=step + "\n", capture_output=True, text=True, timeout=300)
        assert p.returncode == 0, p.stderr[-1500:]
        got[len(ffn)] = (out / "0.f32").read_bytes()
    assert len(got[0]) == len(got[2]) == 2 * 256 * 4 and got[0] != got[2]
