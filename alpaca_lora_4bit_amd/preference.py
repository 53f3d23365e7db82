"""Training on pairs of answers: log-probabilities of the tokens of answers and the loss that prefers one answer of a pair to the other (paired log
ratios against a reference, sigmoid loss).

The reference trains on next tokens only (finetune.py:126-180 of it).  The model that a pair's log ratios are taken against is the same model
with its adapters switched off (`adapters_off`), so no second set of weights is needed.

In a captured graph both functions have their forward and backward pass in one capture, on leaves that no living eager graph holds (torch's accumulation of a
leaf's gradient stays on the stream that it was made on, and a capture that meets another stream ends the process).
"""
import contextlib

import torch

from . import quant_hip


def shifted_labels(labels):
    """labels [B, S] of the tokens themselves -> [B, S] of the tokens that the logits at each place predict: one place to the left, the last place none."""
    moved = torch.full_like(labels, -100, memory_format=torch.contiguous_format)
    moved[..., :-1] = labels[..., 1:]
    return moved


def token_logps(logits, labels):
    """fp32 of labels' shape: log softmax(logits)[label] for logits [..., V] (fp16, bf16 or fp32, any strides) and int64 labels [...], differentiable
    in logits.  A label that is not one of 0 .. V - 1 (-100) is no token: 0, without a gradient.  Logits at a place are those of the token that
    labels has there (`shifted_labels`)."""
    return quant_hip._training().token_logps_autograd(logits, labels)


def preference_loss(logits, labels, ref_logps, beta=0.1, label_smoothing=0.0):
    """(loss [], rewards [2P]) for logits [2P, S, V], int64 labels [2P, S] as for `token_logps` and ref_logps fp32 [2P, S], what `token_logps` gave for the
    reference; sequence p is preferred to sequence p + P.  With r the sums of the answers' log-probabilities less the reference's and z = beta (r[:P] - r[P:])

        loss = mean of -(1 - label_smoothing) log sigmoid(z) - label_smoothing log sigmoid(-z)        rewards = beta r

    differentiable in logits (loss only).  beta > 0, 0 <= label_smoothing <= 0.5."""
    return quant_hip._training().preference_loss_autograd(logits, labels, ref_logps, float(beta), float(label_smoothing))


@contextlib.contextmanager
def adapters_off(model):
    """Within it the model computes without its LoRA adapters (Linear4bitLt's, and those of peft's own layers beside them) and as in evaluation: with dropout
    of its own every pass of a reference would be another one.  Each layer gets its own state back afterwards, each module its own mode and each parameter of a layer its own
    requires_grad.  A model without adapters is refused."""
    layers = [(m, m.disable_adapters) for m in model.modules() if hasattr(m, "lora_A") and hasattr(m, "enable_adapters")]
    if not layers:
        raise ValueError("the model has no LoRA adapters to switch off: it would be its own reference")
    training = [m for m in model.modules() if m.training]
    trained = [(p, p.requires_grad) for layer, _ in layers for p in layer.parameters()]      # peft's own switch sets it too
    try:
        for m in training:
            m.training = False
        for layer, _ in layers:
            layer.enable_adapters(False)
        yield model
    finally:
        for layer, off in layers:
            layer.enable_adapters(not off)
        for p, wanted in trained:
            p.requires_grad_(wanted)
        for m in training:
            m.training = True
