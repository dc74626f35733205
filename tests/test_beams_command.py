"""Beams from the command line."""
import pytest

import dunelix_cases as D
import zirunex_cases as C
from popxl_addons_b200 import generate
from popxl_addons_b200.models import registry
from test_beams import MODEL, generator

PROMPTS = [[5, 17, 3], [8, 2, 9, 4]]


@pytest.fixture
def folder(tmp_path):
    C.write_model(tmp_path, MODEL, C.checkpoint(MODEL, 8))
    return str(tmp_path)


def lines(capsys, folder, *more):
    args = [x for p in PROMPTS for x in ("--prompt", " ".join(map(str, p)))]
    assert generate.main(["--model", folder, *args, "--max-new-tokens", "6", "--dtype", "float32", "--device", "cpu", *more]) == 0
    return [[int(x) for x in line.split()] for line in capsys.readouterr().out.splitlines()]


@pytest.mark.parametrize("prompts,options", [("auto", {}), ("copied", {}), ("shared", {"shared_prefixes": True})])
def test_best_beams_are_printed(folder, capsys, prompts, options):
    gen = generator(("cpu", "float32"), C.checkpoint(MODEL, 8), batch=6, options=options, beams=3, max_new_tokens=6)
    want = [b[0].tokens.tolist() for b in gen.generate_beams(PROMPTS, 6, 7, 0.8)]
    assert lines(capsys, folder, "--beams", "3", "--end", "7", "--length-penalty", "0.8", "--prefixes", prompts) == want


def test_the_model_holds_prompts_once(folder, capsys, monkeypatch):
    """What the command line makes of the choice and of the sizes."""
    made, load = [], registry.load_model
    monkeypatch.setattr(registry, "load_model", lambda *a, **kw: made.append(kw["model_options"]) or load(*a, **kw))
    for more, want in ((["--prefixes", "shared"], {"shared_prefixes": True}), ([], {}), (["--cache", "int8"], {"cache": "int8"})):
        lines(capsys, folder, "--beams", "2", *more)
        assert made.pop() == want
    auto = dict(choice="auto", model=folder, dtype="bfloat16", cache="model", beams=8, positions=generate.SHARED_FROM)
    assert generate.shares_prompts(**auto)
    for other in (dict(choice="copied"), dict(dtype="float32"), dict(cache="int8"), dict(beams=1), dict(positions=generate.SHARED_FROM - 1)):
        assert not generate.shares_prompts(**(auto | other))


def test_models_without_shared_prefixes(tmp_path):
    cfg = next(iter(D.CASES.values()))
    D.write_model(tmp_path, cfg, D.checkpoint(cfg))
    assert not generate.shares_prompts("auto", str(tmp_path), "bfloat16", "model", 8, 1 << 20)
    assert "shared_prefixes" in registry.architecture("Zirunex").options() and registry.architecture("GPT-2").options() == ()


def test_refusals(folder):
    for more in (["--prefixes", "shared"], ["--end", "3"], ["--beams", "2", "--prefixes", "both"]):
        with pytest.raises(SystemExit):
            generate.main(["--model", folder, "--prompt", "5", *more])
    with pytest.raises(ValueError, match="shared"):
        generate.main(["--model", folder, "--prompt", "5", "--device", "cpu", "--beams", "2", "--prefixes", "shared", "--cache", "int8"])


def test_prompts_without_a_continuation(tmp_path, capsys):
    """A model whose logits are no numbers leaves no beam: an empty line for each prompt."""
    ckpt = {k: v * float("nan") if k.endswith("mix.o") else v for k, v in C.checkpoint(MODEL, 8).items()}
    C.write_model(tmp_path, MODEL, ckpt)
    assert lines(capsys, str(tmp_path), "--beams", "3") == [[], []]
