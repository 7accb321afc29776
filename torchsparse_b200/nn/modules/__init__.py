from .activation import *
from .bev import *
from .conv import *
from .embedding import *
from .norm import *
from .tensor_ops import *
