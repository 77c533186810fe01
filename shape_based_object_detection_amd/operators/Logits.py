"""Logits before a label is chosen: penalties for repeated labels, biases, masks.

What suppresses repeated answers of a detector that answers label by label, as ``iou_utils.nms`` suppresses
repeated boxes (the reference has neither such detectors nor this).  ROCm tensors run one HIP kernel
(``sbod_logits_process``), CPU tensors the host path.
"""
from .. import core
from .. import hostpath
from ..metrics import on_host


def process_logits(logits, history=None, history_len=None, prompt_len=None, repetition=1.0, presence=0.0,
                   frequency=0.0, bias=None, bias_ids=None, bias_values=None, allowed=None, out=None):
    """Logits [N, V] (or [V]) as a decoder is to see them; a new tensor, or ``out`` (which may be ``logits``).

    In this order, in 32 bits with one rounding at the end:

    * a label of the row's history: ``x / repetition`` where x > 0, else ``x * repetition``;
    * a label of the answered part, count times: ``- frequency * count - presence`` (infinite ones forbid it);
    * ``+ bias`` ([V] or [N, V], float32 or the logits' type), ``+ bias_values`` (float32) at ``bias_ids``
      ([M] or [N, M], M <= 4096; a label listed twice adds both);
    * ``-inf`` where ``allowed`` forbids the label: truth values [V] or [N, V], or int32 words [W] or [N, W]
      with label v in bit ``v % 32`` of word ``v // 32``.  A forbidden label is -inf whatever it was before;
      a row that allows nothing is all -inf.

    ``history`` [N, L] (or [L]: the same for every row; L < 2^29) int32 / int64: its first ``history_len`` [N] entries count
    (default: all), the first ``prompt_len`` [N] of them were given (repetition only), the others answered.
    ``repetition`` (> 0), ``presence``, ``frequency``: numbers, or float tensors [N].  An id outside [0, V) is
    absent (padding).  Not differentiable: tensors that require a gradient are refused while gradients are on, and
    ones with a forward-mode tangent.
    """
    r = core.label_call('label_logits', logits, logits, history, history_len, prompt_len, repetition, presence, frequency,
                        bias, bias_ids, bias_values, allowed, out)
    if r is not None:
        return r
    args = core.logits_arguments(logits, history, history_len, prompt_len, repetition, presence, frequency, bias,
                                 bias_ids, bias_values, allowed, out)
    if on_host(*[t for t in args if hasattr(t, 'is_cuda')]):
        return hostpath.process_logits(*args)
    return core.process_logits(*args)
