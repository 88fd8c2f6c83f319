"""Hot ops: hand-written gfx950 HIP kernels (GPU) with PyTorch fp32 oracles (CPU)."""
from .conv import ConvGeom, conv2d, conv_fwd, conv_dgrad, conv_wgrad, same_padding
from .bn import batch_norm_act
from .pool import max_pool2d, global_avg_pool
from .loss import softmax_cross_entropy, confidence_penalty_cross_entropy, lovasz_hinge
from .logprob import label_log_probs, LabelLogProbs
from .dropout import dropout, DropoutKeys
from .int8 import int8_linear, quantize_rows, Int8Rows, Int8Weight
from .dwconv import depthwise_conv2d, laplace
from .upsample import upsample as upsample_bilinear_tf1
from .elementwise import add_relu, relu, add, sigmoid_threshold
from .metrics import seg_scores, StreamingMean, IOU_THRESHOLDS
from . import optim

__all__ = ["ConvGeom", "conv2d", "conv_fwd", "conv_dgrad", "conv_wgrad", "same_padding",
           "batch_norm_act", "max_pool2d", "global_avg_pool", "softmax_cross_entropy",
           "confidence_penalty_cross_entropy",
           "lovasz_hinge", "label_log_probs", "LabelLogProbs", "dropout", "DropoutKeys",
           "int8_linear", "quantize_rows", "Int8Rows", "Int8Weight",
           "depthwise_conv2d", "laplace", "upsample_bilinear_tf1", "add_relu", "relu", "add",
           "sigmoid_threshold", "seg_scores", "StreamingMean", "IOU_THRESHOLDS", "optim"]
