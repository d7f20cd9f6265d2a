"""Sizes that the GPT app's generation refuses before it does anything on a device (so without a GPU too)."""
import pytest

from test_gpt_paged import run_app, tokens_file, write_case

SMALL = ["--layers", 1, "--dmodel", 64, "--heads", 1, "--vocab", 32, "--ctx", 16]


@pytest.mark.parametrize("more", [[], ["--beams", 2], ["--budget", 8]], ids=["greedy", "beams", "bounded"])
@pytest.mark.parametrize("name", ["--new", "--prompt", "--batch", "--vocab"])
def test_nothing_to_generate(name, more):
    sizes = {"--prompt": 4, "--new": 4, "--batch": 2, "--vocab": 32, name: 0}
    args = [x for kv in sizes.items() for x in kv]
    assert "at least 1" in run_app("generate", *SMALL[:6], "--ctx", 16, *args, *more, ok=False)


@pytest.mark.parametrize("sizes", [("--prompt", 12, "--new", 5), ("--prompt", 4, "--new", -1), ("--prompt", -1, "--new", 2)])
def test_longer_than_the_context(sizes):
    for more in ([], ["--beams", 2]):
        assert "exceed the context" in run_app("generate", *SMALL, *sizes, *more, ok=False)


def test_beam_check(tmp_path):
    write_case(tmp_path, 1, 32, 1, 12, 20, 2)
    tokens_file(tmp_path, 20, 2, 12)
    for sizes in (("--new", 0), ("--new", -1), ("--prompt", 0), ("--prompt", 8, "--new", 5)):
        assert "need 1 <= prompt" in run_app("beam-check", tmp_path, "cpu", *sizes, ok=False)
