"""Sample from a checkpoint: ``python -m nexttransformer_b200.generate --checkpoint DIR --prompt TEXT``.

``--batch FILE`` answers every line of FILE at once through the paged cache (dense models and delta-rule
hybrids); a penalty or bias option does the same for the one prompt.
"""
import argparse
from pathlib import Path

import torch


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__)
    p.add_argument("--checkpoint", type=Path, required=True)
    p.add_argument("--tokenizer", type=Path, help="directory with tokenizer.pkl")
    p.add_argument("--prompt", default="")
    p.add_argument("--tokens", type=int, default=64)
    p.add_argument("--temperature", type=float, default=1.0)
    p.add_argument("--top-k", type=int, default=50)
    p.add_argument("--seed", type=int, default=42)
    p.add_argument("--no-cache", action="store_true")
    p.add_argument("--batch", type=Path, help="one prompt a line, answered together")
    p.add_argument("--repetition-penalty", type=float, help="divides positive, multiplies negative logits of seen tokens")
    p.add_argument("--presence-penalty", type=float, help="subtracted once from tokens of the answer")
    p.add_argument("--frequency-penalty", type=float, help="subtracted for each occurrence in the answer")
    p.add_argument("--bias", default="", help="TOKEN:VALUE,... added to logits")
    p.add_argument("--stop", type=int, action="append", default=[], help="token that ends an answer (repeatable)")
    a = p.parse_args(argv)
    from nexttransformer_b200.inference import generate, generate_batch
    from nexttransformer_b200.models import load_model
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    model, _ = load_model(a.checkpoint, dev)
    model.eval()
    if a.tokenizer:
        from nexttransformer_b200.runtime.tokenizer import BPETokenizer
        tok = BPETokenizer.from_directory(a.tokenizer)
    options = dict(repetition=a.repetition_penalty, presence=a.presence_penalty, frequency=a.frequency_penalty,
                   bias={int(k): float(v) for k, v in (e.split(":") for e in a.bias.split(",") if e)} or None)
    if a.batch or any(v is not None for v in options.values()) or a.stop:
        lines = a.batch.read_text().splitlines() if a.batch else [a.prompt]
        prompts = [tok.encode(line, prepend=tok.get_bos_token_id()) if a.tokenizer else [int(t) for t in line.split()] or [0]
                   for line in lines]
        for ids, out in zip(prompts, generate_batch(model, prompts, a.tokens, a.temperature, a.top_k, a.seed, a.stop,
                                                    **options)):
            print(tok.decode(ids + out) if a.tokenizer else " ".join(map(str, out)))
        return
    if a.tokenizer:
        ids = tok.encode(a.prompt, prepend=tok.get_bos_token_id())
        out = list(generate(model, ids, a.tokens, a.temperature, a.top_k, a.seed, not a.no_cache))
        print(tok.decode(ids + out))
    else:
        ids = [int(t) for t in a.prompt.split()] or [0]
        print(" ".join(str(t) for t in generate(model, ids, a.tokens, a.temperature, a.top_k, a.seed,
                                                 not a.no_cache)))


if __name__ == "__main__":
    main()
