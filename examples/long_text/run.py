"""Train a small decoder on texts longer than its attention window, score a text
with it, sharpen it with a policy step, and let it answer past the texts' length:

    python examples/long_text/run.py [--device cuda:0 --steps 40]

The texts repeat a short random phrase, so a model that looks back one phrase
predicts them. Window attention (with the first tokens as sinks), residual
dropout, token log probabilities and the key-value ring are all on the path."""

from __future__ import annotations

import argparse
import os
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.dirname(os.path.dirname(HERE)))


def texts(B, n, period, vocab, seed, device):
    import torch

    g = torch.Generator()
    g.manual_seed(seed)
    phrase = torch.randint(1, vocab, (B, period), generator=g)
    return phrase.repeat(1, n // period + 2)[:, :n + 1].to(device)


def main(argv=None) -> int:
    import torch

    from elysium_wan_b200 import ops
    from elysium_wan_b200.models.config import make_config
    from elysium_wan_b200.models.decode import Decoder
    from elysium_wan_b200.models.gpt import StageModel
    from elysium_wan_b200.runtime import optim

    ap = argparse.ArgumentParser()
    ap.add_argument("--device", default="cuda:0" if torch.cuda.is_available() else "cpu")
    ap.add_argument("--steps", type=int, default=400)
    ap.add_argument("--seq", type=int, default=96)
    ap.add_argument("--answer", type=int, default=120)
    a = ap.parse_args(argv)
    cuda = a.device.startswith("cuda")
    dt = "bf16" if cuda else "fp32"
    period, vocab, B = 7, 64, 8
    cfg = make_config("llama_tiny", n_layer=2, vocab_size=vocab, seq_len=a.seq, attn_window=24,
                      attn_sinks=2, dropout=0.05, compute_dtype=dt, boundary_dtype=dt)
    model = StageModel(cfg, (0, cfg.n_entries), a.device, seed=1)
    st = model.store
    opt = optim.build("adamw", st.master, st.grad, st.work, 1e-3,
                      {"betas": (0.9, 0.95), "eps": 1e-8, "weight_decay": 0.0})

    def backward(saved, dl=None):
        if dl is not None:  # another objective than the mean cross-entropy
            saved[-1][1]["dl"] = dl
        tasks: list = []
        model.backward(saved, None, tasks)
        for t in tasks:
            t.run()
        opt.step()
        model.after_step()

    losses = []
    for step in range(a.steps):
        t = texts(B, a.seq, period, vocab, step, a.device)
        model.zero_grad()
        loss, saved = model.forward(t[:, :-1].contiguous(), t[:, 1:].contiguous(), draw=step)
        backward(saved)
        losses.append(float(loss))
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f}")

    # scoring: how sure is it of each token, and of what else?
    dec = Decoder(model)
    t = texts(2, a.seq, period, vocab, 10_000, a.device)
    r = dec.score(t[:, :-1], t[:, 1:], top=3)
    late = r.logp.view(2, a.seq)[:, 2 * period:]
    print(f"mean log probability of a repeated token {late.mean():.3f}, entropy "
          f"{r.entropy.view(2, a.seq)[:, 2 * period:].mean():.3f}, best token right "
          f"{(r.top_ids[:, 0] == t[:, 1:].reshape(-1)).float().mean():.2f}")

    # one policy step: raise the sampled tokens' log probability and the entropy
    x, y = t[:, :-1].contiguous(), t[:, 1:].contiguous()
    model.zero_grad()
    _, saved = model.forward(x, y)
    lg = dec._logits_of(saved[-1][1]["h"])
    s = ops.token_logprobs(lg, vocab, y.reshape(-1))
    n = y.numel()
    weight = torch.full((n,), -1.0 / n, device=a.device)  # minimised: minus the mean log probability
    dl = ops.token_logprobs_bwd(lg, vocab, y.reshape(-1), s.lse, s.entropy, weight, 0.01 * weight)
    backward(saved, dl)

    # answers: the ring holds 26 rows a layer, the answers run past seq_len
    lengths = torch.tensor([a.seq, a.seq // 2], dtype=torch.int32, device=a.device)
    caches = dec.new_caches(2)
    pos = dec.prefill(t[:, :-1], lengths, caches)
    want = texts(2, 2 * a.seq + a.answer, period, vocab, 10_000, a.device)
    tok = want.gather(1, pos[:, None])[:, 0]  # the first token after each prompt
    right = 0
    for i in range(a.answer):
        out = dec.step(tok, pos, caches, top=1)
        tok, pos = out.top_ids[:, 0], pos + 1
        right += int((tok == want.gather(1, pos[:, None])[:, 0]).sum())
    print(f"answered {a.answer} tokens twice, {right / (2 * a.answer):.2f} as the text goes on")
    return 0 if losses[-1] < losses[0] else 1


if __name__ == "__main__":
    sys.exit(main())
