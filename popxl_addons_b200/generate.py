"""Generation from a model folder, greedy or by beam search: `python -m popxl_addons_b200.generate --model DIR --prompt "5 17 3" --prompt "8"`.
Prompts are token ids; one line of token ids is printed per prompt (with `--beams`, the best continuation's)."""
import argparse
import sys

__all__ = ["main"]

# Positions of all beams' prompts from which on it pays to hold a prompt once. A step's attention of 16 heads on 4, us copied / shared: 8 x 4 beams behind
# 1000 positions 24 / 27, behind 4000 60 / 41; 16 x 8 behind 200 25 / 35, behind 1000 63 / 36; 1 x 8 behind 4000 23 / 38, behind 16000 57 / 52.
SHARED_FROM = 1 << 16


def shares_prompts(choice: str, model: str, dtype: str, cache: str, beams: int, positions: int) -> bool:
    """Whether a prompt's beams share its positions, which all of them together hold `positions` times. `choice`: "shared", "copied" or "auto": from
    `SHARED_FROM` on, where the model can and the kernels of 16 bits run."""
    from .models.registry import load_config

    if choice != "auto" or beams < 2 or cache != "model" or dtype != "bfloat16" or positions < SHARED_FROM:
        return choice == "shared"
    return "shared_prefixes" in load_config(model)[0].options()


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(prog="popxl_addons_b200.generate", description="Generation from token ids.")
    ap.add_argument("--model", required=True, help="folder with config.json and model.safetensors")
    ap.add_argument("--prompt", action="append", required=True, help="token ids separated by spaces or commas; repeatable")
    ap.add_argument("--max-new-tokens", type=int, default=32)
    ap.add_argument("--dtype", default="bfloat16", choices=("bfloat16", "float32"))
    ap.add_argument("--batch", type=int, default=0, help="sequences run together (default: all prompts, at most 16)")
    ap.add_argument("--max-seq", type=int, default=0, help="positions a sequence can hold (default: what the prompts need)")
    ap.add_argument("--device", default="auto")
    ap.add_argument("--cache", default="model", choices=("model", "int8"), help="how keys and values are held (int8: where the architecture offers it)")
    ap.add_argument("--repetition-penalty", type=float, default=1.0)
    ap.add_argument("--frequency-penalty", type=float, default=0.0)
    ap.add_argument("--presence-penalty", type=float, default=0.0)
    ap.add_argument("--beams", type=int, default=0, help="beam search with so many beams per prompt (default: greedy)")
    ap.add_argument("--end", type=int, default=None, help="with --beams: the token that ends a continuation")
    ap.add_argument("--length-penalty", type=float, default=0.0, help="with --beams: sums are divided by the number of tokens to this power")
    ap.add_argument("--prefixes", default="auto", choices=("auto", "shared", "copied"),
                    help="with --beams: whether a prompt's beams share its keys and values or have a copy each (default: by their number)")
    a = ap.parse_args(argv)
    if not a.beams and (a.end is not None or a.length_penalty or a.prefixes != "auto"):
        ap.error("--end, --length-penalty and --prefixes belong to --beams")
    from .models.registry import load_model
    from .models.sequence_generator import LogitShaping

    prompts = [[int(x) for x in p.replace(",", " ").split()] for p in a.prompt]
    shaping = LogitShaping(a.repetition_penalty, a.frequency_penalty, a.presence_penalty)
    need = max(len(p) for p in prompts) + a.max_new_tokens
    batch = a.batch or min(len(prompts), 16)
    options = {} if a.cache == "model" else {"cache": a.cache}
    if shares_prompts(a.prefixes, a.model, a.dtype, a.cache, a.beams, batch * a.beams * max(len(p) for p in prompts)):
        options["shared_prefixes"] = True
    gen = load_model(a.model, dtype=a.dtype, batch=batch * max(1, a.beams), max_seq=a.max_seq or need, max_new_tokens=a.max_new_tokens,
                     device=a.device, shaping=shaping != LogitShaping(), beams=a.beams, model_options=options)
    shaping = shaping if gen.shaping else None
    if a.beams:
        out = [beams[0].tokens if beams else () for beams in gen.generate_beams(prompts, a.max_new_tokens, a.end, a.length_penalty, shaping)]
    else:
        out = gen.generate(prompts, a.max_new_tokens, shaping)
    for row in out:
        print(" ".join(str(int(x)) for x in row))
    return 0


if __name__ == "__main__":
    sys.exit(main())
