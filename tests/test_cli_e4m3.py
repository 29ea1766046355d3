"""The command line's options for feed-forwards in 8 bits: what they refuse, without a GPU."""
import json

import pytest

import harness as H  # noqa: F401  (path setup)
from tiny_configs import TINY_A

from lastengine_b200.cli import main


def test_8_bits_beside_32_are_refused_in_words(tmp_path):
    p = tmp_path / "config.json"
    p.write_text(json.dumps(TINY_A))
    with pytest.raises(SystemExit, match="lastengine generate: .*bfloat16 engine, not float32"):
        main(["generate", "--config", str(p), "--prompt-ids", "1,2,3", "--dtype", "float32", "--ffn-dtype", "e4m3"])
