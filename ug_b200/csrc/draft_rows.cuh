// What the operators on drafted nodes share.
#pragma once
#include "ugb_internal.h"

constexpr int UGB_TREE_MAX = 128;    // nodes of a sequence's tree, and nodes that can be kept of it
