"""Distillation from a teacher's top logits on the HIP kernels `ur_distill_forward / _backward`: a loss, with its gradient, for
scores over many classes (candidate poses, views of a grid) whose teacher is known for a few classes per row only -- the
candidates that were rendered, with their errors as logits, or the top logits another network left.

    distill_top_logits(logits, teacher_logits, teacher_index, temperature=1.0, reduction="mean")

p = softmax(teacher_logits / T) over a row's filled slots, q = softmax(logits / T) over all classes (last dimension);
a row's loss is T^2 * sum_j p_j (log p_j - log q[index_j]).  A slot with a negative index is empty (what `route_candidates`
leaves where nothing was eligible); several slots may name one class; a row without a filled slot has loss and gradient
0 and does not count in the mean.  The teacher gets no gradient.  A class index beyond the logits makes its row NaN, as
a NaN among the row's logits or teacher logits does; -inf rules a class or slot out (a class the teacher wants
that the student rules out makes the loss infinite, its gradient stays finite).  The student's sum is float32, so a
row's loss is off by about 1e-7 T^2: at a large T it says little where the loss itself does not grow with T^2 (a teacher that
knows every class).
"""
import torch

from . import native

MAX_SLOTS = 1024
REDUCTIONS = {"none": native.REDUCE_NONE, "sum": native.REDUCE_SUM, "mean": native.REDUCE_MEAN}


def distill_top_logits(logits, teacher_logits, teacher_index, temperature=1.0, reduction="mean"):
    """logits (..., V); teacher_logits, teacher_index (..., k) with the same leading dimensions.  -> float32: one value, or
    one per row with reduction="none"."""
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits need a last dimension of at least 1, got shape {tuple(logits.shape)}")
    native.check_type(logits, "logits")
    native.check_type(teacher_logits, "teacher_logits")
    if teacher_index.dtype is not torch.int64 and teacher_index.dtype is not torch.int32:
        raise ValueError(f"teacher_index must be int32 or int64, got {teacher_index.dtype}")
    if teacher_logits.dim() < 1 or teacher_logits.shape != teacher_index.shape or teacher_logits.shape[-1] < 1 \
            or teacher_logits.shape[:-1] != logits.shape[:-1]:
        raise ValueError(f"teacher_logits and teacher_index must have shape {tuple(logits.shape[:-1])} + (k,), got "
                         f"{tuple(teacher_logits.shape)} and {tuple(teacher_index.shape)}")
    if teacher_logits.shape[-1] > MAX_SLOTS:
        raise NotImplementedError(f"at most {MAX_SLOTS} teacher slots, got {teacher_logits.shape[-1]}")
    if reduction not in REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(REDUCTIONS)}, got {reduction!r}")
    temperature = float(temperature)
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError(f"temperature must be between 1e-30 and 1e30, got {temperature}")
    teacher_logits = teacher_logits.detach().contiguous()
    teacher_index = teacher_index.contiguous()
    native.on_gpu(logits)
    return native.nodes().distill(logits, teacher_logits, teacher_index, temperature, REDUCTIONS[reduction])
