"""Rules on logits in front of the choice of a token: penalties for repeated tokens, biases by token, a grammar's mask.

    apply_rules   the logits under the rules, and each row's best token
    Rules         what a decoder applies at every step

The reference leaves these to its caller (test/nvidia/module/opt/modeling_opt_ours.py:1229 returns the lm_head's logits);
nothing here has a counterpart there.
"""
import torch

import quant


def apply_rules(logits, ids=None, lengths=None, generated_from=None, repetition=None, presence=None, frequency=None, bias_ids=None,
                bias=None, mask=None, out=None, token=None):
    """logits fp16 or fp32 [M, V] -> (logits under the rules, of the same type; the best token of each row, int64 [M]).

    ids int64 [M, L] (any strides), the rows' texts, lengths int64 [M] tokens of each that count (None: all L), the generated
    part from place generated_from int64 [M] on (None: all of it is).  repetition, presence, frequency fp32 [M] or None;
    bias_ids int32 and bias fp32 [M, N]; mask int32 [M or 1, ceil(V / 32)], bit i % 32 of word i / 32 for token i.  In this order,
    each step in fp32:

        x / repetition where x > 0, x * repetition elsewhere    tokens of the text
        x - frequency * c, x - presence                          tokens that stand c > 0 times in the generated part
        x + bias                                                 tokens that bias_ids names (the last entry of several counts)
        -inf                                                     tokens whose bit is 0

    Ids outside the vocabulary are none.  The best token is that of the returned logits: the lowest among equals; NaN never
    wins, and where all are NaN the token is 0.  Where none is above -inf it is the lowest that is -inf, which may be one that
    the mask forbids: the row has no token that may be chosen.  out (which may be logits, or apart from them) and token receive the results where they
    are given.  All on the device and read by the kernels, so that a captured HIP graph follows them."""
    got = quant.logit_rules(logits, ids, lengths, generated_from, repetition, presence, frequency, bias_ids, bias, mask, out, token)
    if got is not None:
        return got if out is None and token is None else (got[0] if out is None else out, got[1] if token is None else token)
    _check(logits, ids, lengths, generated_from, repetition, presence, frequency, bias_ids, bias, mask, out, token)
    # what cannot be read as it lies is copied
    given = [None if x is None else x.contiguous() for x in (repetition, presence, frequency, bias_ids, bias, mask)]
    rows = logits if logits.stride(1) == 1 or logits.shape[1] == 1 else logits.contiguous()
    got = quant.logit_rules(rows, ids, lengths, generated_from, *given, out, token)
    if got is None:
        raise ValueError("rules on logits %s: too large, or out overlaps them in another place" % (tuple(logits.shape),))
    return got if out is None and token is None else (got[0] if out is None else out, got[1] if token is None else token)


def _check(logits, ids, lengths, generated_from, repetition, presence, frequency, bias_ids, bias, mask, out, token):
    if logits.dim() != 2 or logits.dtype not in (torch.float16, torch.float32) or not logits.is_cuda or logits.shape[1] < 1:
        raise ValueError("logits must be fp16 or fp32 [rows, vocabulary] on the device, got %s %s on %s"
                         % (logits.dtype, tuple(logits.shape), logits.device))
    m, v = logits.shape

    def check(name, x, dtype, *shape):
        if x is not None and (x.dtype != dtype or x.dim() != len(shape) or x.device != logits.device
                              or any(n is not None and n != g for n, g in zip(shape, x.shape))):
            raise ValueError("%s must be %s %s on the device of the logits, got %s %s on %s"
                             % (name, dtype, ["any" if n is None else n for n in shape], x.dtype, tuple(x.shape), x.device))

    check("ids", ids, torch.int64, m, None)
    check("lengths", lengths, torch.int64, m)
    check("generated_from", generated_from, torch.int64, m)
    for name, x in (("repetition", repetition), ("presence", presence), ("frequency", frequency)):
        check(name, x, torch.float32, m)
        if x is not None and ids is None:
            raise ValueError("%s is for the tokens of a text; pass ids" % name)
    if (bias_ids is None) != (bias is None):
        raise ValueError("bias_ids and bias come together")
    check("bias_ids", bias_ids, torch.int32, m, None)
    if bias is not None:
        check("bias", bias, torch.float32, m, bias_ids.shape[1])
        if bias.shape[1] > 65535:
            raise ValueError("%d biases a row; 65535 are the most" % bias.shape[1])
    if mask is not None:
        check("mask", mask, torch.int32, 1 if mask.dim() and mask.shape[0] == 1 else m, (v + 31) // 32)
    check("out", out, logits.dtype, m, v)
    if out is not None and ((v > 1 and out.stride(1) != 1) or (m > 1 and out.stride(0) < v)):
        raise ValueError("out must have adjacent elements in rows that lie apart, got strides %s" % (out.stride(),))
    check("token", token, torch.int64, m)
    if token is not None and not token.is_contiguous():
        raise ValueError("token must be contiguous")


class Rules:
    """What `apply_rules` is given at every step of a batch, all but the texts (OPTDecoder.greedy_step): tensors on the device,
    which may be changed in place between the steps, as a grammar's mask is."""

    def __init__(self, repetition=None, presence=None, frequency=None, generated_from=None, bias_ids=None, bias=None, mask=None):
        self.repetition, self.presence, self.frequency, self.generated_from = repetition, presence, frequency, generated_from
        self.bias_ids, self.bias, self.mask = bias_ids, bias, mask

    def penalises(self):
        """Whether the texts count: one of the penalties is given."""
        return any(x is not None for x in (self.repetition, self.presence, self.frequency))

    def apply(self, logits, ids=None, lengths=None, out=None, token=None):
        if not self.penalises():
            ids = lengths = None  # nobody asks for the texts
        return apply_rules(logits, ids, lengths, self.generated_from if ids is not None else None, self.repetition, self.presence,
                           self.frequency, self.bias_ids, self.bias, self.mask, out, token)
