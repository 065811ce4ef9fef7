"""Logit controls (guidance, repetition / presence / frequency penalties, biases, masks) in 64 bits on the CPU: the definition behind
mv_op_logit_controls.  No reference counterpart."""
import numpy as np


def controls(logits, uncond=None, guidance=None, repetition=None, presence=None, frequency=None, history=None, history_len=None, prompt_len=None,
             bias_ids=None, bias=None, masks=None, mask_index=None):
    """Arrays as mv_logit_controls has them (bias_ids / bias with one row: for all rows) -> out [rows][vocab], allowed [rows], size [rows][vocab]:
    the magnitudes that enter an element, for error bounds."""
    rows, vocab = logits.shape
    out = logits.astype(np.float64).copy()
    size = np.abs(out)
    allowed = np.full(rows, vocab, dtype=np.int64)
    with np.errstate(invalid="ignore", over="ignore"):
        for r in range(rows):
            x, s = out[r], size[r]
            if uncond is not None:
                g = float(guidance[r])
                # an infinite logit, a guidance of 1, and beyond 1 a token that the unconditioned row excludes: x stays
                live = ~(np.isinf(x) | (g == 1) | ((uncond[r] == -np.inf) & (g > 1)))
                s[live] = np.abs(g * x[live]) + np.abs((1 - g) * uncond[r][live])
                x[live] = g * x[live] + (1 - g) * uncond[r][live]
            if history is not None:
                n = history.shape[1] if history_len is None else min(max(int(history_len[r]), 0), history.shape[1])
                p = 0 if prompt_len is None else int(prompt_len[r])
                rho = 1.0 if repetition is None else float(repetition[r])
                count, seen = np.zeros(vocab), np.zeros(vocab, dtype=bool)
                for i, t in enumerate(history[r, :n].tolist()):
                    if 0 <= t < vocab:
                        seen[t] = True
                        count[t] += i >= p
                x[seen] = np.where(x[seen] > 0, x[seen] / rho, x[seen] * rho)
                s[seen] *= max(rho, 1 / rho, 1.0)
                off = count * (0.0 if frequency is None else float(frequency[r])) + (count > 0) * (0.0 if presence is None else float(presence[r]))
                x -= off
                s += np.abs(off)
            if bias_ids is not None:
                b = r if bias_ids.shape[0] > 1 else 0
                for t, v in {t: v for t, v in zip(bias_ids[b].tolist(), bias[b].tolist()) if 0 <= t < vocab}.items():
                    x[t] += v
                    s[t] += abs(v)
            if masks is not None:
                m = r if mask_index is None else int(mask_index[r])
                if 0 <= m < masks.shape[0]:
                    ok = ((masks[m].astype(np.uint32)[:, None] >> np.arange(32, dtype=np.uint32)) & 1).reshape(-1)[:vocab].astype(bool)
                    x[~ok] = -np.inf
                    allowed[r] = int(ok.sum())
    return out, allowed, size
